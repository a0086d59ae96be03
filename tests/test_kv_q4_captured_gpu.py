"""Captured attention steps over the cache in 4 bits whose sequences grow far beyond what they were captured with."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc
from test_kv_q4_gpu import Mirror, _dev, held

pytestmark = pytest.mark.gpu
GPU = "cuda"


class Captured:
    """Both layers' attention of one step in a graph, on buffers of `room` tokens."""

    def __init__(self, ctx, m, room, batch):
        self.ctx, self.m = ctx, m
        self.stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
        t = torch.bfloat16 if m.dtype == "bf16" else torch.float32
        self.rows = [[torch.zeros(room, h, m.hd, device=GPU, dtype=t) for h in (m.heads, m.n_kv, m.n_kv)] for _ in range(m.layers)]
        self.out = [torch.full((room, m.heads, m.hd), -7.0, device=GPU, dtype=t) for _ in range(m.layers)]
        m.cache.batch(*batch)
        ctx.synchronize()
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            for layer, ((q, k, v), out) in enumerate(zip(self.rows, self.out)):
                m.cache.attend_dev(layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), m.hd ** -0.5, out.data_ptr())

    def step(self, rng, seqs, pos0, counts):
        m, T = self.m, sum(counts)
        new = [m.rows(rng, T) for _ in range(m.layers)]
        m.cache.batch(seqs, pos0, counts)
        for layer in range(m.layers):
            for to, x in zip(self.rows[layer], new[layer]):
                to[:T].copy_(_dev(x, m.dtype))
            self.out[layer].fill_(-7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(self.stream):
            self.graph.replay()
        self.ctx.synchronize()
        for layer, (q, k, v) in enumerate(new):
            at, got = 0, self.out[layer].float().cpu().numpy()
            for s, p, n in zip(seqs, pos0, counts):
                for store, x in ((m.k[layer], k), (m.v[layer], v)):
                    store[s] = np.concatenate([store.get(s, np.zeros((0, m.n_kv, m.hd), np.float32))[:p], held(x[at:at + n])])
                m.compare(got[at:at + n], q[at:at + n], s, p, m.hd ** -0.5, layer)
                at += n
            assert np.all(got[at:] == -7.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64)])
def test_replays_go_on_where_the_plan_outgrows_its_room(ctx, dtype, heads, kv, hd):
    """From 300 positions past 384, where a sequence is first split, past 1000 and 5000, with a prompt of another sequence in between, whose plan is far larger."""
    rng = np.random.default_rng(hd)
    m = Mirror(ctx, dtype, heads, kv, hd, 3, 420, layers=2)
    a, b, c = (m.cache.seq_alloc() for _ in range(3))

    def fill(seqs, pos0, counts):
        for layer in range(2):
            m.step(rng, seqs, pos0, counts, layer=layer, check=False)

    fill([a, b], [0, 0], [300, 90])
    g = Captured(ctx, m, 6, ([a, b], [300, 90], [1, 1]))
    for i in range(2):
        g.step(rng, [a, b], [300 + i, 90 + i], [1, 1])
    fill([a, b], [302, 92], [81, 1])
    for i in range(3):
        g.step(rng, [a, b], [383 + i, 93 + i], [1, 1])
    fill([c], [0], [1500])
    g.step(rng, [a, c, b], [386, 1500, 96], [1, 3, 2])      # more entries and tokens than it was captured with
    fill([a], [387], [700])
    g.step(rng, [a, b], [1087, 98], [1, 1])
    fill([a], [1088], [4000])
    for i in range(2):
        g.step(rng, [b, a, c], [99 + i, 5088 + i, 1503 + i], [1, 1, 1])
    g.step(rng, [b], [40], [1])                             # and back to less
    # a second capture on the grown plan, in turn with the first
    h = Captured(ctx, m, 3, ([a, b], [5090, 41], [1, 2]))
    for i in range(2):
        h.step(rng, [a, b], [5090 + 2 * i, 41 + 3 * i], [1, 2])
        g.step(rng, [a, b], [5091 + 2 * i, 43 + 3 * i], [1, 1])
    del g.graph, h.graph


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_writes_alone(ctx, dtype):
    rng = np.random.default_rng(3)
    m = Mirror(ctx, dtype, 4, 2, 64, 2, 200)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    m.step(rng, [a], [0], [10], check=False)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = (torch.zeros(900, 2, 64, device=GPU, dtype=t) for _ in "kv")
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    m.cache.batch([a], [10], [1])
    ctx.synchronize()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        m.cache.write_dev(0, k.data_ptr(), v.data_ptr())
    for seqs, pos0, counts in (([a], [10], [1]), ([b, a], [0, 11], [880, 20]), ([a, b], [31, 880], [1, 2])):
        rows = m.rows(rng, sum(counts))
        m.cache.batch(seqs, pos0, counts)
        for to, x in zip((k, v), rows[1:]):
            to[:len(x)].copy_(_dev(x, dtype))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        at = 0
        for s, p, n in zip(seqs, pos0, counts):
            for store, x in ((m.k[0], rows[1]), (m.v[0], rows[2])):
                store[s] = np.concatenate([store.get(s, np.zeros((0, 2, 64), np.float32))[:p], held(x[at:at + n])])
            m.check_blocks(s)
            at += n
    del graph


def test_a_step_that_a_capture_does_not_serve_leaves_cache_and_results(ctx):
    """Prompt-sized entries beside a decoded token: rows behind those of the captured call are not read, nothing is written, and the status says so."""
    rng = np.random.default_rng(4)
    m = Mirror(ctx, "bf16", 8, 2, 128, 2, 40)
    a, b = m.cache.seq_alloc(), m.cache.seq_alloc()
    m.step(rng, [a, b], [0, 0], [100, 30])
    q, k, v = (torch.full((60, h, 128), 3.0, device=GPU, dtype=torch.bfloat16) for h in (8, 2, 2))
    out = torch.full_like(q, -7.0)
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    m.cache.batch([b, a], [30, 100], [1, 1])
    ctx.synchronize()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        m.cache.attend_dev(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0.1, out.data_ptr())
    m.cache.batch([b, a], [30, 100], [1, 40])
    half = torch.full((41, 2, 128), 0.5, device=GPU, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    m.cache.write_dev(0, half.data_ptr(), half.data_ptr())
    ctx.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    with pytest.raises(dc.DcError) as e:
        ctx.synchronize()
    assert e.value.status == -6 and torch.all(out == -7.0)
    for s, p, n in ((b, 30, 1), (a, 100, 40)):
        for store in (m.k[0], m.v[0]):
            store[s] = np.concatenate([store[s], np.full((n, 2, 128), 0.5, np.float32)])
        m.check_blocks(s)
    rows = m.rows(rng, 2)
    m.cache.batch([b, a], [31, 140], [1, 1])
    for to, x in zip((q, k, v), rows):
        to[:2].copy_(_dev(x, "bf16"))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    ctx.synchronize()
    for i, (s, p) in enumerate(((b, 31), (a, 140))):
        for store, x in ((m.k[0], rows[1]), (m.v[0], rows[2])):
            store[s] = np.concatenate([store[s], held(x[i:i + 1])])
        m.compare(out[i:i + 1].float().cpu().numpy(), rows[0][i:i + 1], s, p, 0.1)
    del graph
