"""Steps whose tokens lie on more pages than one launch takes (slots times pages that a sequence's new tokens may lie on beyond 16384): lengths, pages, tables and places against the simulation."""
import numpy as np
import pytest
import torch

from kv_dev_util import Steps, ints, stream_of

pytestmark = pytest.mark.gpu
ALL = 2**31 - 1


class Pair:
    def __init__(self, ctx, slots, pages, a_slot, max_tokens):
        self.kv, self.want = ctx.kv_cache_dev(1, 1, 1, 64, pages, slots, a_slot, max_tokens), Steps(slots, pages, a_slot, max_tokens)

    def step(self, count, drop, most):
        c, d = ints(count), ints(drop)
        torch.cuda.synchronize()
        self.kv.step_dev(c.data_ptr(), drop=d.data_ptr(), max_count=most)
        self.want.step(np.asarray(count).tolist(), np.asarray(drop).tolist(), most)
        self.want.check(self.kv)


@pytest.mark.parametrize("slots,a_slot", [(512, 64), (300, 200), (4096, 6)])
def test_large_steps(ctx, slots, a_slot):
    """Admissions, drops with fewer and with more pages asked for than freed, a pool that runs out, a step with tokens enough; small steps on the pages that large ones freed."""
    rng = np.random.default_rng(slots)
    most, zero, all_ = 16 * a_slot, np.zeros(slots, int), np.full(slots, ALL)
    pages, tokens = slots * a_slot * 2 // 3, slots * most // 2
    assert slots * min(most // 16 + 2, a_slot) > 16384
    p = Pair(ctx, slots, pages, a_slot, tokens)
    p.step(rng.integers(0, most // 2, slots), zero, most)                              # from nothing
    p.step(rng.integers(0, 6, slots), rng.integers(0, 4, slots), 5)                    # a small one
    p.step(rng.integers(0, most // 8, slots), all_, most)                              # fewer pages than freed
    assert len(p.want.stack) > pages // 2
    p.step(rng.integers(0, 6, slots), zero, 5)                                         # (on pages that the large one freed)
    p.step(rng.integers(most // 4, most // 2, slots), rng.integers(0, most // 8, slots), most)      # more than freed
    p.step(rng.integers(0, most + 2, slots), zero, most)                               # the pool, tables and tokens run out
    assert 0 < sum(c == 0 for c in p.want.counts) < slots
    p.step(rng.integers(0, 6, slots), rng.integers(0, 40, slots), 5)
    p.step(rng.integers(0, most, slots) * (rng.random(slots) < 0.5), np.where(rng.random(slots) < 0.5, ALL, 0), most)
    p.step(rng.integers(-3, most + 40, slots), np.where(rng.random(slots) < 0.3, ALL, rng.integers(-9, most, slots)), most)
    p.step(zero, all_, most)                                                           # all end
    assert p.want.lens == [0] * slots and len(p.want.stack) == pages
    p.step(np.full(slots, most // 3), zero, most)
    p.step(np.full(slots, 3), zero, 3)
    p.kv.close()


def test_tokens_of_a_step_run_out(ctx):
    p = Pair(ctx, 512, 512 * 64, 64, 100000)
    for _ in range(3):
        p.step(np.full(512, 700), np.full(512, ALL), 1024)
        assert 0 < sum(p.want.counts) <= 100000 and p.want.counts[-1] == 0
    p.kv.close()


def test_one_sequence_of_a_million_tokens(ctx):
    p = Pair(ctx, 3, 84000, 82000, 1310000)
    p.step([0, 1300000, 0], [0, 0, 0], 1300000)
    p.step([70, 5, 9], [0, 0, 0], 70)
    p.step([300000, 0, 17], [0, 600001, 0], 300000)
    p.step([1, 1, 1], [ALL, 3, 0], 1)
    p.step([0, 1000000, 1300000], [0, ALL, ALL], 1310000)
    p.kv.close()


def test_small_steps_that_free_many_pages(ctx):
    """Long sequences that end in a step of single tokens."""
    p = Pair(ctx, 512, 512 * 64, 64, 512 * 1024)
    p.step(np.full(512, 1000), np.zeros(512, int), 1024)
    p.step(np.arange(512) % 2, np.where(np.arange(512) % 3, ALL, 0), 1)
    p.step(np.arange(512) % 2, np.full(512, ALL), 1)
    p.kv.close()


def test_captured_large_steps(ctx):
    slots, a_slot = 512, 64
    kv, want = ctx.kv_cache_dev(1, 1, 1, 64, 20000, slots, a_slot, 300000), Steps(slots, 20000, a_slot, 300000)
    rng = np.random.default_rng(5)
    count, drop = ints(np.zeros(slots)), ints(np.zeros(slots))
    torch.cuda.synchronize()
    kv.step_dev(count.data_ptr(), drop=drop.data_ptr(), max_count=1000)
    ctx.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), stream_of(ctx)
    with torch.cuda.graph(graph, stream=stream):
        kv.step_dev(count.data_ptr(), drop=drop.data_ptr(), max_count=1000)
    for _ in range(5):
        c, d = rng.integers(0, 1001, slots), np.where(rng.random(slots) < 0.5, ALL, rng.integers(0, 400, slots))
        count.copy_(ints(c)), drop.copy_(ints(d))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        want.step(c.tolist(), d.tolist(), 1000)
        want.check(kv)
    kv.close()
