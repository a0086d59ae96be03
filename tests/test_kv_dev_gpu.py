"""A paged cache of 16-bit rows whose sequences are kept on the GPU: steps against a simulation, attention against 64 bits."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc
from kv_dev_util import GPU, Mirror, Steps, ints, stream_of

pytestmark = pytest.mark.gpu
ALL = 2**31 - 1


# ------------------------------------------------------------------------------------------------ steps
@pytest.mark.parametrize("slots,pages,a_slot,max_tokens,most", [(1, 4, 4, 64, 20), (7, 12, 5, 40, 30), (33, 100, 9, 300, 40), (1025, 3000, 6, 20000, 60), (4096, 5000, 3, 9000, 9)])
def test_steps_of_lengths_pages_and_tables(ctx, slots, pages, a_slot, max_tokens, most):
    """Random steps, most of which ask for more than there is: drops beyond a sequence's length, counts below 0 and above the step's or the table's limit, pages and tokens that run out."""
    rng = np.random.default_rng(slots)
    kv = ctx.kv_cache_dev(1, 1, 1, 64, pages, slots, a_slot, max_tokens)
    want = Steps(slots, pages, a_slot, max_tokens)
    for i in range(12):
        count = rng.integers(-1 if i % 3 == 2 else 0, most + 3, slots) * (rng.random(slots) < (0.3 if i % 2 else 0.9))
        drop = np.where(rng.random(slots) < 0.15, ALL, rng.integers(-2, 2 * most, slots) * (rng.random(slots) < 0.5))
        c, d = ints(count), ints(drop)
        torch.cuda.synchronize()
        kv.step_dev(c.data_ptr(), drop=d.data_ptr(), max_count=most)
        want.step(count.tolist(), drop.tolist(), most)
        want.check(kv)
    kv.close()


def test_a_step_and_the_one_that_takes_it_back(ctx):
    """Tables and the pool are as they were, whoever got pages from whom; what lies behind a step's tokens stays."""
    rng = np.random.default_rng(3)
    kv, want = ctx.kv_cache_dev(1, 1, 1, 64, 400, 40, 20, 6400), Steps(40, 400, 20, 6400)
    a, b, grow = rng.integers(1, 160, 40), rng.integers(1, 160, 40), rng.integers(1, 20, 40)
    zero, all_ = np.zeros(40, int), np.full(40, ALL)

    def step(count, drop, most):
        c, d = ints(count), ints(drop)
        torch.cuda.synchronize()
        kv.step_dev(c.data_ptr(), drop=d.data_ptr(), max_count=most)
        want.step(count.tolist(), drop.tolist(), most)
        want.check(kv)
    step(a, zero, 160)
    tables, stack = [list(t) for t in want.tables], list(want.stack)
    for _ in range(2):
        step(b, all_, 160)
        step(a, all_, 160)
        assert want.tables == tables and want.stack == stack
        step(grow, zero, 20)
        behind = kv.read("slots")[int(grow.sum()):]
        step(zero, grow, 0)
        assert want.tables == tables and want.stack == stack and np.array_equal(kv.read("slots")[int(grow.sum()):], behind)
    kv.close()


def test_steps_without_arrays(ctx):
    kv, want = ctx.kv_cache_dev(1, 2, 1, 64, 8, 3, 4, 64), Steps(3, 8, 4, 64)
    count = ints([5, 17, 0])
    torch.cuda.synchronize()
    kv.step_dev(count.data_ptr(), max_count=17)
    want.step([5, 17, 0], [0] * 3, 17)
    want.check(kv)
    kv.step_dev(0, max_count=3)
    want.step([0] * 3, [0] * 3, 3)
    want.check(kv)
    kv.step_dev(0, drop=count.data_ptr(), max_count=0)
    want.step([0] * 3, [5, 17, 0], 0)
    want.check(kv)
    kv.close()


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [(1, 1, 64), (8, 8, 128), (6, 2, 128), (12, 1, 64), (32, 4, 128), (24, 4, 64), (40, 1, 128), (5, 5, 64), (18, 2, 64)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_attention_of_steps(ctx, dtype, heads, kv, hd):
    """Single tokens, drafted ones and prompts of sequences from nothing to some hundred positions, some left out, over all positions and over windows."""
    m = Mirror(ctx, dtype, heads, kv, hd, 6, 400, 60, 700, seed=heads)
    for count, drop, window, keep in (([1, 5, 0, 16, 33, 200], None, 0, 0), ([1, 1, 1, 1, 1, 1], None, 0, 0), ([3, 0, 5, 2, 1, 4], [0, 2, 0, 7, 0, 30], 0, 0), ([1, 1, 0, 1, 1, 1], None, 17, 0),
                                      ([2, 3, 4, 1, 5, 2], [1, 1, 1, 1, 1, 1], 40, 5), ([1] * 6, None, 1, 0), ([1] * 6, None, 64, 100), ([30, 0, 64, 1, 9, 100], None, 50, 20),
                                      ([0, 0, 0, 0, 1, 0], None, 0, 0), ([70, 2, 1, 0, 3, 17], [0, 0, ALL, ALL, 0, 0], 16, 16)):
        m.step(count, drop)
        m.steps.check(m.cache)
        m.attend(window=window, keep=keep)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_long_sequences_shared_out(ctx, dtype):
    """Lengths of which many CTAs have a part, beside short ones; then drafted tokens at all offsets of a page."""
    m = Mirror(ctx, dtype, 8, 2, 128, 5, 1400, 700, 16000, seed=5)
    m.step([9000, 1, 3000, 40, 0])
    T = len(m.steps.seqs)
    k, v = m.rows(T, 2), m.rows(T, 2)
    kd, vd = k.to(GPU), v.to(GPU)
    torch.cuda.synchronize()
    m.cache.write_dev(0, kd.data_ptr(), vd.data_ptr())
    m.ctx.synchronize()
    m.append(0, k, v)
    for i, (window, keep) in enumerate(((0, 0), (0, 0), (2000, 4), (100, 0), (5000, 3000))):
        m.step([1, 1, 1, 1, 1] if i % 2 else [5, 2, 7, 16, 3])
        m.attend(window=window, keep=keep)


@pytest.mark.parametrize("n", [33, 70, 1025])
def test_many_sequences(ctx, n):
    """More sequences than a warp looks at at once, one in three without new tokens."""
    m = Mirror(ctx, "bf16", 4, 2, 64, n, 3 * n + 8, 40, 8 * n, seed=n)
    m.step([(7 * s) % 8 if s % 3 else 0 for s in range(n)])
    m.attend()
    m.step([(s % 2) * (1 + s % 3) for s in range(n)])
    m.attend()
    m.step([1] * n)
    m.attend(window=5, keep=2)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift", [((8, 8, 8), (0, 0, 0)), ((3, 5, 1), (0, 0, 0)), ((0, 0, 0), (1, 1, 1)), ((2, 2, 2), (3, 2, 5)), ((0, 4, 0), (0, 4, 2))])
def test_strides_and_alignments(ctx, dtype, pad, shift):
    for hd in (64, 128):
        m = Mirror(ctx, dtype, 6, 2, hd, 3, 40, 12, 200, seed=7)
        m.step([40, 3, 90])
        m.attend(pad=pad, shift=shift)
        m.step([1, 4, 1])
        m.attend(pad=pad, shift=shift)
        m.step([2, 2, 40])
        m.attend(pad=pad, shift=shift, written=True, window=30, keep=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_that_the_cache_holds(ctx, dtype, hd):
    """What attention writes and what the writing call writes: the rows as they are, f32 ones as fp16, in two layers."""
    m = Mirror(ctx, dtype, 6, 3, hd, 3, 30, 12, 300, layers=2, seed=11)
    for i, count in enumerate(([21, 100, 3], [1, 2, 0], [40, 0, 16], [5, 1, 1])):
        m.step(count)
        m.attend(0)
        m.attend(1, written=True)
    for layer in range(2):
        for s in range(3):
            for at in range(m.steps.lens[s]):
                k, v = m.cache.read_page(layer, m.steps.tables[s][at // 16]) if at % 16 == 0 else (k, v)
                for x, want in ((k, m.k[layer][s]), (v, m.v[layer][s])):
                    x = (x.astype(np.uint32) << 16).view(np.float32) if dtype == "bf16" else x
                    assert np.array_equal(x[at % 16].astype(np.float64), want[at])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_and_nan_reach_those_that_see_them_alone(ctx, dtype):
    """A value that is no number reaches its head's later tokens of its sequence, as long as it is in sight; nothing else."""
    m = Mirror(ctx, dtype, 8, 2, 64, 3, 60, 20, 500, seed=13)
    m.step([40, 37, 20])
    T = len(m.steps.seqs)
    k, v = m.rows(T, 2), m.rows(T, 2)
    v[33, 0, 5] = float("nan")          # position 33 of sequence 0: not seen by its first 33 tokens
    v[40 + 3, 1, 60] = float("inf")     # position 3 of sequence 1
    k[40 + 20, 1, 9] = float("nan")
    m.attend(k=k, v=v, window=12, keep=2)
    for _ in range(3):
        m.step([5, 8, 1])
        m.attend(window=12, keep=2)     # the bad rows move out of sight
    m.step([70, 1, 1])
    m.attend(window=20)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_full_of_nan_are_used_again(ctx, dtype):
    """Places of a page behind a sequence's end hold whatever was there."""
    m = Mirror(ctx, dtype, 8, 2, 128, 2, 10, 10, 200, seed=17)
    m.step([150, 0])
    bad = torch.full((150, 2, 128), float("nan")).to(m.rows(1, 1).dtype)
    b = bad.to(GPU)
    torch.cuda.synchronize()
    m.cache.write_dev(0, b.data_ptr(), b.data_ptr())
    m.step([3, 37], [ALL, ALL])
    m.attend()
    m.step([5, 60], [0, 0])
    m.attend()
    m.step([1, 1], [0, 20])
    m.attend(window=4)


def test_scores_of_any_size(ctx):
    """Queries and keys from 1e-4 to hundreds, scales of both signs and 0: weights on one key, on all alike, and with a rising maximum."""
    for dtype in ("f32", "bf16", "f16"):
        m = Mirror(ctx, dtype, 4, 2, 64, 2, 40, 20, 320, seed=19)
        m.step([200, 100])
        m.attend(q=m.rows(300, 4, 30.0), k=m.rows(300, 2, 20.0))
        for scale, size in ((0.125, 1e-4), (-0.125, 3.0), (0.0, 1.0), (0.125, 100.0), (1.0, 1.0)):
            m.step([2, 1])
            m.attend(q=m.rows(3, 4, size), scale=scale)
        m.step([20, 1])
        m.attend(q=m.rows(21, 4, 1.0), k=m.rows(21, 2) * torch.arange(1, 22)[:, None, None].to(m.rows(1, 1).dtype))


def test_results_are_the_same_every_time(ctx):
    """Parts of a sequence are joined in their order, whoever comes last."""
    m = Mirror(ctx, "bf16", 16, 2, 128, 3, 700, 300, 6000, seed=23)
    m.step([4000, 20, 900])
    T = 4920
    rows = [m.rows(T, h).to(GPU) for h in (16, 2, 2)]
    torch.cuda.synchronize()
    m.cache.write_dev(0, rows[1].data_ptr(), rows[2].data_ptr())
    one = ints([1, 4, 2])
    torch.cuda.synchronize()
    m.cache.step_dev(one.data_ptr(), max_count=4)
    first = None
    for _ in range(20):
        out = torch.zeros(7, 16, 128, dtype=torch.bfloat16, device=GPU)
        torch.cuda.synchronize()
        m.cache.attend_dev(0, rows[0].data_ptr(), rows[1].data_ptr(), rows[2].data_ptr(), 0.09, out.data_ptr())
        m.ctx.synchronize()
        first = out if first is None else first
        assert torch.equal(out, first)


# ------------------------------------------------------------------------------------------------ captured calls, errors
def test_captured_steps_grow(ctx):
    """A graph of a step and its attention, replayed while the sequences grow from nothing over many pages, with drops and counts of its own every time."""
    m = Mirror(ctx, "bf16", 8, 2, 128, 4, 300, 100, 64, seed=29)
    count, drop = ints([0] * 4), ints([0] * 4)
    q, k, v = (torch.zeros(20, h, 128, dtype=torch.bfloat16, device=GPU) for h in (8, 2, 2))
    out = torch.zeros(20, 8, 128, dtype=torch.bfloat16, device=GPU)
    torch.cuda.synchronize()
    m.cache.step_dev(count.data_ptr(), max_count=5)      # (a graph finds its kernels set up)
    m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.1, out.data_ptr(), window=100, keep_first=4)
    ctx.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), stream_of(ctx)
    with torch.cuda.graph(graph, stream=stream):
        m.cache.step_dev(count.data_ptr(), drop=drop.data_ptr(), max_count=5)
        m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.1, out.data_ptr(), window=100, keep_first=4)
    rng = np.random.default_rng(1)
    for i in range(60):
        c, d = rng.integers(0, 6, 4).tolist(), rng.integers(0, 3, 4).tolist()
        count.copy_(ints(c)), drop.copy_(ints(d))
        m.steps.step(c, d, 5)
        T = len(m.steps.seqs)
        new = [m.rows(T, h) for h in (8, 2, 2)]
        for to, x in zip((q, k, v), new):
            to[:T].copy_(x)
        out.fill_(-7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        for rows in (m.k[0], m.v[0]):
            for s in range(4):
                rows[s] = rows[s][:m.steps.lens[s] - m.steps.counts[s]]
        m.append(0, new[1], new[2])
        m.steps.check(m.cache)
        assert (out[T:] == -7).all()
        m.compare(out[:T].cpu(), new[0], 0, 100, 4, 0.1)
    assert max(m.steps.lens) > 64


def test_a_captured_call_reports_a_step_that_is_more_than_its_own(ctx):
    """Attention captured for single tokens that is replayed behind a step with a prompt: its sequence is left alone, and the next synchronisation says so."""
    m = Mirror(ctx, "bf16", 8, 2, 64, 2, 40, 20, 300, seed=31)
    m.step([10, 10])
    m.attend()
    m.step([1, 1])
    q, k, v = (torch.zeros(300, h, 64, dtype=torch.bfloat16, device=GPU) for h in (8, 2, 2))
    out = torch.full((300, 8, 64), -7.0, dtype=torch.bfloat16, device=GPU)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), stream_of(ctx)
    with torch.cuda.graph(graph, stream=stream):
        m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.1, out.data_ptr())
    m.step([200, 1])
    with torch.cuda.stream(stream):
        graph.replay()
    with pytest.raises(dc.DcError, match="more new tokens"):
        ctx.synchronize()
    ctx.synchronize()
    assert (out[:200] == -7).all() and not (out[200] == -7).any()


def test_calls_that_are_refused(ctx):
    kv = ctx.kv_cache_dev(2, 8, 2, 64, 10, 4, 5, 64)
    with pytest.raises(dc.DcError, match="no step yet"):
        kv.attend_dev(0, 256, 256, 256, 0.1, 256)
    kv.step_dev(0, max_count=2)
    for bad in (dict(layer=2), dict(layer=-1), dict(q=0), dict(out=0), dict(k=0), dict(ld_q=511), dict(ld_kv=127), dict(ld_out=3), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1),
                dict(keep_first=3), dict(window=4, keep_first=-1), dict(q=257)):
        a = {**dict(layer=0, q=256, k=256, v=256, scale=0.1, out=256), **bad}
        with pytest.raises(dc.DcError):
            kv.attend_dev(**a)
    with pytest.raises(dc.DcError):
        kv.step_dev(0, max_count=-1)
    with pytest.raises(dc.DcError):
        kv.write_dev(0, 0, 256)
    other = dc.Context(0)
    try:
        with pytest.raises(dc.DcError, match="another context"):
            other._check(dc._lib.lib().dc_b200_kv_step_dev(other.handle, kv.handle, None, None, 1))
    finally:
        other.close()
    from densecore_b200.ops import KVCache
    with pytest.raises(dc.DcError, match="kept on the GPU"):
        KVCache.seq_alloc(kv)
    kv.close()


def test_pages_far_into_a_large_cache(ctx):
    """Offsets beyond 2^32 bytes within a layer, and a second layer behind it."""
    m = Mirror(ctx, "bf16", 16, 8, 128, 3, 84000, 82000, 1310000, layers=2, seed=37)      # 64 KB a page and layer
    m.step([0, 1300000, 0])
    m.step([70, 0, 9], [0, 0, 0])
    assert min(m.steps.slots) // 16 * 65536 > 2**32
    m.attend(1)
    m.attend(0)
    m.step([1, 0, 5])
    m.attend(0)
    m.attend(1, window=30, keep=3)
    m.cache.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_captured_prompt_step(ctx, dtype):
    """Prompts, drafted and single tokens of one graph, replayed on other mixtures of them: portions that are split over their keys, whole tiles, windows."""
    m = Mirror(ctx, dtype, 8, 2, 64, 3, 900, 300, 900, seed=41)
    room = 900
    count, drop = ints([0] * 3), ints([0] * 3)
    t = m.rows(1, 1).dtype
    q, k, v = (torch.zeros(room, h, 64, dtype=t, device=GPU) for h in (8, 2, 2))
    out = torch.zeros(room, 8, 64, dtype=t, device=GPU)

    def call():
        m.cache.step_dev(count.data_ptr(), drop=drop.data_ptr(), max_count=600)
        m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.11, out.data_ptr(), window=700, keep_first=20)
    torch.cuda.synchronize()
    call()
    ctx.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), stream_of(ctx)
    with torch.cuda.graph(graph, stream=stream):
        call()
    for c, d in (([600, 1, 17], [0, 0, 0]), ([1, 300, 5], [0, 0, 3]), ([600, 200, 64], [1, 1, 1]), ([0, 0, 0], [0, 0, 0]), ([1, 1, 1], [0, 0, 0]), ([33, 600, 0], [0, 0, ALL]), ([500, 1, 129], [40, 5, 0])):
        count.copy_(ints(c)), drop.copy_(ints(d))
        m.steps.step(c, d, 600)
        T = len(m.steps.seqs)
        new = [m.rows(T, h) for h in (8, 2, 2)]
        for to, x in zip((q, k, v), new):
            to[:T].copy_(x)
        out.fill_(-7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        for rows in (m.k[0], m.v[0]):
            for s in range(3):
                rows[s] = rows[s][:m.steps.lens[s] - m.steps.counts[s]]
        m.append(0, new[1], new[2])
        m.steps.check(m.cache)
        assert (out[T:] == -7).all()
        m.compare(out[:T].cpu(), new[0], 0, 700, 20, 0.11)


def test_prompts_behind_long_sequences(ctx):
    """Few tiles of rows, so that their keys are split over CTAs and added up, beside single tokens; all the keys or a window of them."""
    for dtype, hd in (("bf16", 128), ("f16", 64)):
        m = Mirror(ctx, dtype, 4, 2, hd, 3, 900, 400, 12000, seed=43)
        m.step([5000, 700, 20])
        T = 5720
        k, v = m.rows(T, 2), m.rows(T, 2)
        kd, vd = k.to(GPU), v.to(GPU)
        torch.cuda.synchronize()
        m.cache.write_dev(0, kd.data_ptr(), vd.data_ptr())
        ctx.synchronize()
        m.append(0, k, v)
        for count, window, keep in (([200, 1, 1], 0, 0), ([40, 3, 300], 0, 0), ([130, 1, 33], 2500, 40), ([65, 200, 0], 0, 0)):
            m.step(count)
            m.attend(window=window, keep=keep)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_near_the_ends_of_their_range(ctx, dtype):
    """Rows from 2^-115 to 2^123 under scales that undo it: results as those of rows around 1."""
    m = Mirror(ctx, dtype, 4, 2, 64, 2, 40, 20, 320, seed=47)
    for power in (-115, 0, 100, 115, 121):
        m.step([1, 70] if power in (0, 115) else [2, 3])
        T = len(m.steps.seqs)
        m.attend(q=m.rows(T, 4) * 2.0**power, scale=64**-0.5 * 2.0**-power)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_more_query_heads_than_a_tile_has_rows(ctx, dtype):
    """A single token has more rows of a key head than the rows kernel takes, or as many, or one fewer."""
    for heads, kv, hd in ((96, 1, 64), (260, 1, 64), (130, 2, 128), (64, 1, 128), (66, 2, 64), (32, 1, 64)):
        m = Mirror(ctx, dtype, heads, kv, hd, 3, 60, 20, 40, seed=53)
        for count, window, keep in (([20, 1, 0], 0, 0), ([1, 1, 1], 0, 0), ([2, 0, 1], 9, 2), ([1, 1, 1], 3, 0)):
            m.step(count)
            m.attend(window=window, keep=keep)
