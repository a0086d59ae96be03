"""The paged cache in 4 bits and attention over it, against the definition in 64 bits.

Rounding that the bounds count: a score is off by at most a (2^-22 of the two fp16 terms of a query + 2^-20 of its sums in f32), a = scale sum |q_i k_i|, and
by 2^-22 of its own size in units of log2 e; a weight by that and 2^-21 of the exponential and the two terms; the answer, a mean of values, by twice the
weights' relative error times the largest value.  bf16 rows: weights p d are rounded to fp16, by 2^-11 of themselves or 2^-25 of the row's largest, and codes d q
reach no further than 2 max |v| (largest less least of a group): 2^-11 (2 max |v|) + n 2^-25 (2 max |v|) for n tokens; results add half a step, eps / 2 relative.  Portions of 64 rows or more (new tokens times query heads of a key head) of bf16 rows take
keys, values and weights as fp16: 2^-11 of a score's sum of magnitudes, and twice 2^-11 max |v|; over a whole result these are of random sign, so that its error's norm
stays below bf16's own 2^-8 of the result's."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc

pytestmark = pytest.mark.gpu
GPU = "cuda"


def held(x):
    """x [..., dim] f32 -> the values that the cache stands for, by the definition's steps."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 64, 64).astype(np.float32)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    m = lo.astype(np.float16).astype(np.float32)
    d = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d > 0, np.clip(np.rint((g - m) / d), 0, 15), 0)
    return (q.astype(np.float64) * d + m).astype(np.float32).reshape(x.shape)


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).bfloat16().float().numpy()


def bits(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).bfloat16().view(torch.uint16).numpy()


def unbits(x):
    return torch.from_numpy(x).view(torch.bfloat16).float().numpy()


def attention(q, K, V, pos0, scale, halves=False):
    """One sequence: q [n, heads, hd], K, V [pos0 + n, kv, hd].  Returns answers and the bound on their error, [n, heads, hd] both."""
    n, heads, hd = q.shape
    G = heads // K.shape[1]
    y, tol = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    for h in range(heads):
        k, v = K[:, h // G].astype(np.float64), V[:, h // G].astype(np.float64)
        for i in range(n):
            c = pos0 + i + 1
            x = q[i, h].astype(np.float64)
            z = scale * (k[:c] @ x)
            a = float(np.abs(scale) * (np.abs(k[:c]) @ np.abs(x)).max())
            w = np.exp(z - z.max())
            y[i, h] = w @ v[:c] / w.sum()
            ds = a * (2.0 ** -22 + 2.0 ** -20 + halves * 2.0 ** -11) + 1.5 * float(np.abs(z).max()) * 2.0 ** -22
            tol[i, h] = (2 * (2 * ds + 2.0 ** -21) + 2.0 ** -20) * np.abs(v[:c]).max()
    return y, tol


class Mirror:
    """A cache on the GPU beside the values that it ought to stand for."""

    def __init__(self, ctx, dtype, heads, kv, hd, seqs, pages, layers=1, blocks=None):
        self.ctx, self.dtype, self.heads, self.n_kv, self.hd = ctx, dtype, heads, kv, hd
        self.cache = ctx.kv_cache_q4(layers, heads, kv, hd, blocks or seqs * pages + 3, seqs, pages, dtype=dtype)
        self.layers = layers
        self.k = [{} for _ in range(layers)]
        self.v = [{} for _ in range(layers)]

    def rows(self, rng, n, spread=1.0):
        out = [rng.normal(size=(n, h, self.hd)).astype(np.float32) * np.float32(s) for h, s in ((self.heads, 1.5), (self.n_kv, spread), (self.n_kv, spread))]
        return [bf16(x) for x in out] if self.dtype == "bf16" else out

    def step(self, rng, seqs, pos0, counts, scale=None, layer=0, rows=None, check=True):
        self.cache.batch(seqs, pos0, counts)
        q, k, v = rows or self.rows(rng, sum(counts))
        scale = scale if scale is not None else self.hd ** -0.5
        wire = bits if self.dtype == "bf16" else (lambda x: x)
        out = self.cache.attend(layer, wire(q), wire(k), wire(v), scale)
        out = unbits(out) if self.dtype == "bf16" else out
        at = 0
        for s, p, n in zip(seqs, pos0, counts):
            for store, new in ((self.k[layer], k), (self.v[layer], v)):
                old = store.get(s, np.zeros((0, self.n_kv, self.hd), np.float32))[:p]
                store[s] = np.concatenate([old, held(new[at:at + n])]) if n else store.get(s, old)
            if check and n:
                self.compare(out[at:at + n], q[at:at + n], s, p, scale, layer)
            at += n
        return out

    def compare(self, out, q, s, p, scale, layer=0):
        halves = self.dtype == "bf16" and len(q) * (self.heads // self.n_kv) >= 64
        y, tol = attention(q, self.k[layer][s], self.v[layer][s], p, scale, halves)
        if halves:
            assert np.linalg.norm(out - y) <= 2.0 ** -8 * np.linalg.norm(y)
        if self.dtype == "bf16":
            v = np.abs(self.v[layer][s]).max()
            tol = tol + 2 * v * (2.0 ** -11 + len(self.v[layer][s]) * 2.0 ** -25)
            tol = tol + (np.abs(y) + tol) * (torch.finfo(torch.bfloat16).eps / 2) + 2.0 ** -126
        assert np.all(np.isfinite(out))
        worst = np.abs(out - y) / tol
        assert worst.max() <= 1.0, (s, p, float(worst.max()), np.unravel_index(worst.argmax(), worst.shape))

    def check_blocks(self, seq, layer=0):
        n = len(self.k[layer][seq])
        for i, b in enumerate(self.cache.block_table(seq)):
            k, v = self.cache.read_block(layer, int(b))
            c = min(16, n - 16 * i)
            if c > 0:
                assert np.array_equal(k[:c], self.k[layer][seq][16 * i:16 * i + c]) and np.array_equal(v[:c], self.v[layer][seq][16 * i:16 * i + c])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,hd", [(1, 1, 128), (16, 8, 128), (32, 4, 128), (6, 2, 64), (24, 4, 64), (16, 1, 128), (12, 1, 64)])
def test_from_the_first_token_on(ctx, dtype, heads, kv, hd):
    """Prompts and single tokens around the pages' ends, three sequences of different lengths at once."""
    rng = np.random.default_rng(heads * 100 + hd)
    m = Mirror(ctx, dtype, heads, kv, hd, 4, 40)
    s = [m.cache.seq_alloc() for _ in range(3)]
    m.step(rng, [s[0]], [0], [1])
    m.step(rng, [s[0], s[1]], [1, 0], [1, 15])
    m.step(rng, [s[1], s[2]], [15, 0], [1, 33])
    m.step(rng, [s[2], s[0], s[1]], [33, 2, 16], [1, 14, 1])
    m.step(rng, s, [16, 17, 34], [1, 1, 1])
    m.step(rng, s[::-1], [35, 18, 17], [200, 3, 0])
    m.step(rng, s, [17, 21, 235], [1, 1, 1])
    for x in s:
        m.check_blocks(x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,context", [(128, 3000), (64, 5001), (128, 12345)])
def test_long_sequences_are_split_and_joined(ctx, dtype, hd, context):
    rng = np.random.default_rng(context)
    m = Mirror(ctx, dtype, 8, 2, hd, 2, context // 16 + 3)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    m.step(rng, [a, b], [0, 0], [context, 77], check=False)
    m.step(rng, [a, b], [context, 77], [1, 1])
    m.step(rng, [b, a], [78, context + 1], [2, 3])


@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 128), (6, 2, 128), (8, 1, 128), (32, 4, 128), (16, 1, 64), (5, 1, 64)])
def test_prompts(ctx, heads, kv, hd):
    """Portions around the sizes of tiles (64 keys, 128 and 256 rows), first ones and later ones, beside decoded tokens and alone."""
    rng = np.random.default_rng(heads + hd)
    m = Mirror(ctx, "bf16", heads, kv, hd, 3, 160)
    a, b, c = (m.cache.seq_alloc() for _ in range(3))
    m.step(rng, [a], [0], [64])
    m.step(rng, [b, a], [0, 64], [257, 1])
    m.step(rng, [c, a, b], [0, 65, 257], [129, 128, 63])
    m.step(rng, [b, c], [320, 129], [1, 300])
    m.step(rng, [a], [193], [90])
    for x in (a, b, c):
        m.check_blocks(x)


@pytest.mark.parametrize("heads,kv,hd,context,count", [(8, 4, 128, 2222, 40), (2, 1, 64, 3001, 70), (16, 2, 128, 1500, 200)])
def test_prompts_behind_long_contexts_are_split(ctx, heads, kv, hd, context, count):
    rng = np.random.default_rng(context)
    m = Mirror(ctx, "bf16", heads, kv, hd, 2, (context + count) // 16 + 2)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    m.step(rng, [a, b], [0, 0], [context, 500], check=False)
    rows = m.rows(rng, count + 1)
    first = m.step(rng, [a, b], [context, 500], [count, 1], rows=rows)
    assert np.array_equal(m.step(rng, [a, b], [context, 500], [count, 1], rows=rows, check=False), first)
    m.step(rng, [b], [501], [32], scale=-0.1)
    m.step(rng, [b], [533], [64], scale=0.0)


def test_a_nan_in_a_prompt_reaches_later_tokens_and_its_group_alone(ctx):
    rng = np.random.default_rng(30)
    m = Mirror(ctx, "bf16", 4, 2, 128, 1, 30)
    a = m.cache.seq_alloc()
    rows = m.rows(rng, 400)
    rows[2][333, 1, 70] = np.nan         # a value: second group of head 1
    rows[1][350, 0, 5] = np.inf          # a key of head 0
    out = m.step(rng, [a], [0], [400], rows=rows, check=False)
    want = np.zeros(out.shape, bool)
    want[333:, 2:, 64:] = True
    want[350:, :2] = True
    assert np.array_equal(np.isnan(out), want)
    k, v = held(rows[1]), held(rows[2])
    y, _ = attention(rows[0][:333], k[:333], v[:333], 0, 128 ** -0.5)
    assert np.linalg.norm(out[:333] - y) <= 2.0 ** -8 * np.linalg.norm(y)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_range_of_values(ctx, dtype):
    """Up to 32768 in magnitude is held, beyond it a group is NaN."""
    rng = np.random.default_rng(31)
    m = Mirror(ctx, dtype, 2, 1, 64, 1, 10)
    a = m.cache.seq_alloc()
    q, k, v = m.rows(rng, 70)
    k[3, 0, :2], v[5, 0, :2] = (32768, -32768), (32768, -32768)
    m.step(rng, [a], [0], [70], rows=(q, k, v), scale=1e-6)
    m.check_blocks(a)
    v[5, 0, 0] = 33024
    out = m.step(rng, [a], [0], [70], rows=(q, k, v), scale=1e-6, check=False)
    assert np.all(np.isnan(out[5:])) and np.all(np.isfinite(out[:5]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_same_step_gives_the_same_bits(ctx, dtype):
    rng = np.random.default_rng(5)
    m = Mirror(ctx, dtype, 32, 4, 128, 2, 400)
    a = m.cache.seq_alloc()
    rows = m.rows(rng, 6000)
    m.step(rng, [a], [0], [6000], rows=rows, check=False)
    one = m.rows(rng, 1)
    first = m.step(rng, [a], [6000], [1], rows=one)
    for _ in range(10):
        assert np.array_equal(m.step(rng, [a], [6000], [1], rows=one, check=False), first)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [1e-6, 1e-4, 1.0, 200.0])
def test_small_and_large_values(ctx, dtype, spread):
    rng = np.random.default_rng(8)
    m = Mirror(ctx, dtype, 4, 2, 128, 1, 30)
    a = m.cache.seq_alloc()
    q, k, v = m.rows(rng, 300, spread)
    m.step(rng, [a], [0], [300], rows=(q, k, v), scale=128 ** -0.5 / spread, check=False)
    q, k, v = m.rows(rng, 2, spread)
    # rows that are constant, zero, or hold one large value
    k[0, 0] = 0.25 * spread
    v[0, 0] = 0
    k[1, 1, :64] = 0
    v[1, 1, 3] = 30 * spread
    if dtype == "bf16":
        k, v = bf16(k), bf16(v)
    m.step(rng, [a], [300], [2], rows=(q, k, v), scale=128 ** -0.5 / spread)
    m.check_blocks(a)


def test_zero_and_huge_scores(ctx):
    """Scale 0: the mean of the values.  One key far above all others: its value."""
    rng = np.random.default_rng(9)
    m = Mirror(ctx, "f32", 2, 1, 64, 1, 20)
    a = m.cache.seq_alloc()
    m.step(rng, [a], [0], [100], scale=0.0)
    q, k, v = m.rows(rng, 1)
    k[0, 0] = 40 * q[0, 0]
    m.step(rng, [a], [100], [1], rows=(q, k, v), scale=1.0)
    m.step(rng, [a], [101], [1], scale=-1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unused_slots_do_not_matter(ctx, dtype):
    """A page that a finished sequence left full of NaN, then taken by another: only written slots are seen."""
    rng = np.random.default_rng(10)
    m = Mirror(ctx, dtype, 4, 2, 128, 2, 8, blocks=8)
    a = m.cache.seq_alloc()
    q, k, v = m.rows(rng, 128)
    bad = [q, np.full_like(k, np.nan), np.full_like(v, np.inf)]
    out = m.step(rng, [a], [0], [128], rows=bad, check=False)
    assert np.all(np.isnan(out))
    kb, vb = m.cache.read_block(0, int(m.cache.block_table(a)[3]))
    assert np.all(np.isnan(kb)) and np.all(np.isnan(vb))
    m.cache.seq_free(a)
    m.k[0].clear(), m.v[0].clear()
    b = m.cache.seq_alloc()
    m.step(rng, [b], [0], [1])
    m.step(rng, [b], [1], [17])
    m.step(rng, [b], [18], [1])
    m.step(rng, [b], [19], [60])


def test_a_nan_stays_with_its_sequence_group_and_later_tokens(ctx):
    rng = np.random.default_rng(11)
    m = Mirror(ctx, "f32", 4, 2, 128, 2, 8)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    rows = m.rows(rng, 40)
    rows[2][25, 1, 70] = np.inf          # sequence a, token 5, head 1, second group of the value
    out = m.step(rng, [b, a], [0, 0], [20, 20], rows=rows, check=False)
    nan = np.isnan(out)
    want = np.zeros_like(nan)
    want[25:, 2:, 64:] = True
    assert np.array_equal(nan, want)
    y, tol = attention(rows[0][:20], held(rows[1])[:20], held(rows[2])[:20], 0, 128 ** -0.5)
    assert np.all(np.abs(out[:20] - y) <= tol)


def test_rewriting_after_a_rollback(ctx):
    """Drafted tokens that were not accepted: the next step starts at an earlier position."""
    rng = np.random.default_rng(12)
    m = Mirror(ctx, "f32", 8, 2, 64, 1, 8)
    a = m.cache.seq_alloc()
    m.step(rng, [a], [0], [30])
    m.step(rng, [a], [30], [5])
    m.step(rng, [a], [32], [5])
    m.step(rng, [a], [0], [3])
    m.step(rng, [a], [3], [1])
    m.check_blocks(a)


def test_forks_share_pages_until_they_write(ctx):
    rng = np.random.default_rng(13)
    m = Mirror(ctx, "bf16", 8, 4, 128, 4, 8, layers=2, blocks=24)
    a = m.cache.seq_alloc()
    for layer in (0, 1):
        m.step(rng, [a], [0], [40], layer=layer)
    free = m.cache.free_blocks()
    b = m.cache.seq_fork(a)
    for layer in (0, 1):
        m.k[layer][b], m.v[layer][b] = m.k[layer][a].copy(), m.v[layer][a].copy()
    assert m.cache.free_blocks() == free
    for layer in (0, 1):
        m.step(rng, [b], [40], [1], layer=layer)
    assert m.cache.free_blocks() == free - 1                       # the third page was copied
    # (every layer's step begins anew at the same positions)
    for layer in (0, 1):
        m.step(rng, [a, b], [40, 41], [2, 1], layer=layer)
    for layer in (0, 1):
        m.check_blocks(a, layer)
        m.check_blocks(b, layer)
    # rewriting an early page of one leaves the other's
    for layer in (0, 1):
        m.step(rng, [b], [5], [4], layer=layer)
        m.step(rng, [a], [42], [1], layer=layer)
        m.check_blocks(a, layer)
        m.check_blocks(b, layer)
    m.cache.seq_free(a)
    m.cache.seq_free(b)
    assert m.cache.free_blocks() == 24


def test_a_prefix_from_the_cache(ctx):
    import ctypes as C
    rng = np.random.default_rng(14)
    m = Mirror(ctx, "f32", 4, 2, 128, 3, 8)
    lib, tokens = dc._lib.lib(), np.arange(50, dtype=np.int32)
    vp = tokens.ctypes.data_as(C.c_void_p)
    a = m.cache.seq_alloc()
    m.step(rng, [a], [0], [50])
    assert lib.dc_b200_kv_prefix_register(m.cache.handle, a, vp, 50) == 0
    b, n = m.cache.seq_alloc(), C.c_int(0)
    assert lib.dc_b200_kv_prefix_attach(m.cache.handle, b, vp, 50, C.byref(n)) == 0 and n.value == 48
    m.k[0][b], m.v[0][b] = m.k[0][a][:48], m.v[0][a][:48]
    m.step(rng, [b], [48], [2])
    m.step(rng, [a, b], [50, 50], [1, 1])
    m.step(rng, [b], [10], [2])          # into a registered page: a copy
    m.step(rng, [a], [51], [1])


def _dev(x, dtype):
    return torch.from_numpy(x).to(GPU, torch.bfloat16 if dtype == "bf16" else torch.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_of_a_fused_projection(ctx, dtype):
    """Rows of one projection [q | k | v | padding] at odd strides and offsets, results into a part of wider rows that stays as it was around them; held values."""
    rng = np.random.default_rng(15)
    heads, kv, hd, T = 6, 2, 64, 21
    m = Mirror(ctx, dtype, heads, kv, hd, 2, 8)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    q, k, v = m.rows(rng, T)
    width = (heads + 2 * kv) * hd + 5
    fused = torch.full((T, width), 9.0, device=GPU, dtype=_dev(q, dtype).dtype)
    base = 3
    fused[:, base:base + heads * hd] = _dev(q, dtype).flatten(1)
    fused[:, base + heads * hd:base + (heads + kv) * hd] = _dev(k, dtype).flatten(1)
    fused[:, base + (heads + kv) * hd:base + (heads + 2 * kv) * hd] = _dev(v, dtype).flatten(1)
    out = torch.full((T + 2, heads * hd + 7), 5.0, device=GPU, dtype=fused.dtype)
    kh, vh = (torch.full((T + 1, kv, hd), 7.0, device=GPU) for _ in "kv")
    torch.cuda.synchronize()
    size = fused.element_size()
    m.cache.batch([a, b], [0, 0], [20, 1])
    at = fused.data_ptr() + base * size
    m.cache.attend_dev(0, at, at + heads * hd * size, at + (heads + kv) * hd * size, hd ** -0.5, out.data_ptr() + size, ld_q=width, ld_kv=width, ld_out=heads * hd + 7,
                       k_held=kh.data_ptr(), v_held=vh.data_ptr())
    ctx.synchronize()
    got = out[:T, 1:1 + heads * hd].float().cpu().numpy().reshape(T, heads, hd)
    rest = out.clone()
    rest[:T, 1:1 + heads * hd] = 5.0
    assert torch.all(rest == 5.0)
    assert np.array_equal(kh[:T].cpu().numpy(), held(k)) and np.array_equal(vh[:T].cpu().numpy(), held(v)) and torch.all(kh[T] == 7) and torch.all(vh[T] == 7)
    for s, lo, n in ((a, 0, 20), (b, 20, 1)):
        m.k[0][s], m.v[0][s] = held(k[lo:lo + n]), held(v[lo:lo + n])
        m.compare(got[lo:lo + n], q[lo:lo + n], s, 0, hd ** -0.5)
    # the rows stand there: attention alone, and writing alone
    again = torch.zeros_like(out)
    torch.cuda.synchronize()
    m.cache.attend_dev(0, at, 0, 0, hd ** -0.5, again.data_ptr() + size, ld_q=width, ld_out=heads * hd + 7)
    m.cache.write_dev(0, at + heads * hd * size, at + (heads + kv) * hd * size, ld=width)
    ctx.synchronize()
    assert torch.equal(again[:T, 1:1 + heads * hd], out[:T, 1:1 + heads * hd])


def test_several_steps_and_caches_in_flight(ctx):
    """Steps of two caches of one context enqueued in turn without waiting: every one sees its own plan."""
    rng = np.random.default_rng(16)
    ms = [Mirror(ctx, "f32", 8, 2, 128, 3, 20) for _ in range(2)]
    seqs = [[m.cache.seq_alloc() for _ in range(3)] for m in ms]
    lens, keep = [[0, 0, 0], [0, 0, 0]], []
    for step in range(12):
        for i, m in enumerate(ms):
            counts = [int(rng.integers(0, 24)) for _ in range(3)]
            q, k, v = m.rows(rng, sum(counts))
            t = [_dev(x, "f32") for x in (q, k, v)]
            out = torch.full_like(t[0], -3.0)
            torch.cuda.synchronize() if step == 0 else torch.cuda.current_stream().synchronize()
            m.cache.batch(seqs[i], lens[i], counts)
            m.cache.attend_dev(0, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), 128 ** -0.5, out.data_ptr())
            keep.append((i, list(lens[i]), counts, q, k, v, t, out))
            lens[i] = [a + c for a, c in zip(lens[i], counts)]
    ctx.synchronize()
    for i, before, counts, q, k, v, _, out in keep:
        m, at, got = ms[i], 0, out.cpu().numpy()
        for s, p, n in zip(seqs[i], before, counts):
            for store, new in ((m.k[0], k), (m.v[0], v)):
                store[s] = np.concatenate([store.get(s, np.zeros((0, 2, 128), np.float32)), held(new[at:at + n])])
            if n:
                m.compare(got[at:at + n], q[at:at + n], s, p, 128 ** -0.5)
            at += n


def test_a_captured_step_replays_on_the_newest_plan(ctx):
    rng = np.random.default_rng(17)
    m = Mirror(ctx, "f32", 8, 2, 128, 2, 40)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    m.step(rng, [a, b], [0, 0], [300, 90])
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    q, k, v = (torch.zeros(2, h, 128, device=GPU) for h in (8, 2, 2))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    m.cache.batch([a, b], [300, 90], [1, 1])
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(dc.DcError):
            m.cache.batch([a, b], [300, 90], [1, 1])
        m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 128 ** -0.5, out.data_ptr())
    for step in range(20):
        rows = m.rows(rng, 2)
        m.cache.batch([a, b], [300 + step, 90 + step], [1, 1])
        ctx.synchronize()
        for to, x in zip((q, k, v), rows):
            to.copy_(torch.from_numpy(x))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for i, (s, p) in enumerate(((a, 300 + step), (b, 90 + step))):
            m.k[0][s], m.v[0][s] = np.concatenate([m.k[0][s], held(rows[1][i:i + 1])]), np.concatenate([m.v[0][s], held(rows[2][i:i + 1])])
            m.compare(out[i:i + 1].cpu().numpy(), rows[0][i:i + 1], s, p, 128 ** -0.5)
    del graph


def test_a_step_without_tokens_is_not_captured(ctx):
    m = Mirror(ctx, "f32", 4, 2, 64, 2, 4)
    a = m.cache.seq_alloc()
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    x = torch.zeros(1, 4, 64, device=GPU)
    torch.cuda.synchronize()
    m.cache.batch([a], [0], [0])
    m.cache.attend_dev(0, x.data_ptr(), x.data_ptr(), x.data_ptr(), 1.0, x.data_ptr())      # nothing to do
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in (lambda: m.cache.attend_dev(0, x.data_ptr(), x.data_ptr(), x.data_ptr(), 1.0, x.data_ptr()),
                     lambda: m.cache.write_dev(0, x.data_ptr(), x.data_ptr())):
            with pytest.raises(dc.DcError) as e:
                call()
            assert e.value.status == -7
    del graph


def test_a_million_new_tokens_at_once(ctx):
    """Caches filled in one step: more tiles than a grid's second dimension holds."""
    n, each = 64, 17000
    m = Mirror(ctx, "bf16", 16, 1, 64, n, -(-each // 16))
    seqs = [m.cache.seq_alloc() for _ in range(n)]
    torch.manual_seed(5)
    q, k, v = (torch.randn(n * each, h, 64, device=GPU, dtype=torch.bfloat16) for h in (16, 1, 1))
    kh, vh = (torch.empty(n * each, 1, 64, device=GPU) for _ in "kv")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    m.cache.batch(seqs, [0] * n, [each] * n)
    m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.125, out.data_ptr(), k_held=kh.data_ptr(), v_held=vh.data_ptr())
    ctx.synchronize()
    for i in (0, n // 2, n - 1):
        rows = slice(i * each, (i + 1) * each)
        new = [bf16(x[rows].float().cpu().numpy()) for x in (k, v)]
        m.k[0][seqs[i]], m.v[0][seqs[i]] = (held(x) for x in new)
        assert np.array_equal(kh[rows].cpu().numpy(), m.k[0][seqs[i]]) and np.array_equal(vh[rows].cpu().numpy(), m.v[0][seqs[i]])
        for p in (0, each // 2, each - 4):
            at = slice(i * each + p, i * each + p + 4)
            y, store = m.k[0][seqs[i]], m.v[0][seqs[i]]
            m.k[0][seqs[i]], m.v[0][seqs[i]] = y[:p + 4], store[:p + 4]
            m.compare(out[at].float().cpu().numpy(), q[at].float().cpu().numpy(), seqs[i], p, 0.125)
            m.k[0][seqs[i]], m.v[0][seqs[i]] = y, store


def test_prompt_sized_portions_are_not_captured(ctx):
    rng = np.random.default_rng(33)
    m = Mirror(ctx, "bf16", 8, 2, 128, 2, 40)
    a = m.cache.seq_alloc()
    m.step(rng, [a], [0], [100])
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    q, k, v = (torch.zeros(40, h, 128, device=GPU, dtype=torch.bfloat16) for h in (8, 2, 2))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    call = lambda: m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 1.0, out.data_ptr())
    m.cache.batch([a], [100], [16])          # 64 rows
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(dc.DcError) as e:
            call()
        assert e.value.status == -7
    m.cache.batch([a], [100], [15])          # 60 rows
    call()
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    m.cache.batch([a], [100], [40])          # a replay on a step that it does not serve is reported
    with torch.cuda.stream(stream):
        graph.replay()
    with pytest.raises(dc.DcError) as e:
        ctx.synchronize()
    assert e.value.status == -6
    m.cache.batch([a], [100], [3])
    with torch.cuda.stream(stream):
        graph.replay()
    ctx.synchronize()
    del graph


def test_refusals(ctx):
    rng = np.random.default_rng(18)
    for bad in (dict(head_dim=96), dict(n_head=3), dict(dtype="f16"), dict(n_layer=0), dict(max_blocks=0)):
        args = dict(n_layer=1, n_head=4, n_kv_head=2, head_dim=128, max_blocks=8, max_seqs=2, max_blocks_per_seq=4, dtype="f32") | bad
        with pytest.raises(dc.DcError):
            ctx.kv_cache_q4(**args)
    m = Mirror(ctx, "f32", 4, 2, 128, 3, 4, blocks=5)
    c = m.cache
    q, k, v = m.rows(rng, 1)

    def refused(status, call, *a, **kw):
        with pytest.raises(dc.DcError) as e:
            call(*a, **kw)
        assert e.value.status == status, e.value

    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256)                # no batch yet
    refused(-1, c.batch, [0], [0], [1])                                  # not allocated
    a, b = c.seq_alloc(), c.seq_alloc()
    refused(-1, c.batch, [a, a], [0, 0], [1, 1])                         # twice
    refused(-1, c.batch, [7], [0], [1])
    refused(-1, c.batch, [a], [1], [1])                                  # a hole
    refused(-1, c.batch, [a], [0], [-1])
    refused(-3, c.batch, [a], [0], [65])                                 # beyond its table
    m.step(rng, [a], [0], [33])                                          # three of five blocks
    refused(-3, c.batch, [a, b], [33, 0], [1, 33])                       # out of blocks: nothing has changed
    assert c.free_blocks() == 2 and len(c.block_table(a)) == 3 and len(c.block_table(b)) == 0
    m.step(rng, [a], [33], [1])
    refused(-1, c.attend_dev, 1, 256, 256, 256, 1.0, 256)                # layer
    refused(-1, c.attend_dev, 0, 0, 256, 256, 1.0, 256)                  # null rows
    refused(-1, c.attend_dev, 0, 256, 256, 0, 1.0, 256)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 0)
    refused(-1, c.attend_dev, 0, 256, 256, 256, float("nan"), 256)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256, ld_q=511)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256, ld_kv=255)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256, ld_out=511)
    refused(-1, c.attend_dev, 0, 256, 0, 0, 1.0, 256, k_held=256)
    refused(-1, c.write_dev, 0, 0, 256)
    # a fork, a free and a lookup end the step
    f = c.seq_fork(a)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256)
    m.k[0][f], m.v[0][f] = m.k[0][a], m.v[0][a]
    m.step(rng, [f], [34], [1])
    c.seq_free(f)
    refused(-1, c.attend_dev, 0, 256, 256, 256, 1.0, 256)
    # a host call that fails leaves zeros
    out = np.full((1, 4, 128), 3.0, np.float32)
    vp = dc.ops._vp
    assert dc._lib.lib().dc_b200_flash_attn_q4(ctx.handle, c.handle, 9, vp(q), vp(k), vp(v), 1.0, vp(out)) == -1
    m.step(rng, [a], [34], [1])
    assert dc._lib.lib().dc_b200_flash_attn_q4(ctx.handle, c.handle, 9, vp(q), vp(k), vp(v), 1.0, vp(out)) == -1 and not out.any()
    # calls of the other cache
    fp16 = ctx.kv_cache(1, 2, 128, 4, 2, 2)
    assert dc._lib.lib().dc_b200_kv_batch(fp16.handle, 0, None, None, None) == -1
    refused(-1, c.flash_attn_decode, 0, q, k, v, [a], [35], 1.0)
    fp16.close()
    # steps without tokens do nothing
    c.batch([], [], [])
    c.attend_dev(0, 0, 0, 0, 1.0, 0)
    c.batch([a, b], [35, 0], [0, 0])
    c.attend_dev(0, 0, 0, 0, 1.0, 0)
    assert c.attend(0, np.zeros((0, 4, 128), np.float32), np.zeros((0, 2, 128), np.float32), np.zeros((0, 2, 128), np.float32), 1.0).shape == (0, 4, 128)
    m.step(rng, [b], [0], [2])
    c.close()
