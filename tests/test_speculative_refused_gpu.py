"""Speculative steps in one CUDA graph over a pool that runs short: a sequence whose tokens a step refuses keeps what it has, gets no tokens, drops nothing in the next step, and is served once
there are pages."""
import numpy as np
import pytest
import torch

from kv_dev_util import GPU, Mirror, ints, stream_of
from test_verify_rows_gpu import check

pytestmark = pytest.mark.gpu
HEADS, KV, HD, V, R, D = 4, 2, 64, 500, 6, 3
ROWS = R * (D + 1)
ALL = 2**31 - 1


@pytest.mark.parametrize("pages,max_tokens", [(9, ROWS), (40, 13)])
def test_refused_sequences_are_left_alone_and_served_later(ctx, pages, max_tokens):
    """Refused for want of pages, or because the step has tokens enough."""
    rng = np.random.default_rng(pages)
    m = Mirror(ctx, "f32", HEADS, KV, HD, R, pages, 6, max_tokens, seed=3)
    a = m.cache.arrays()
    assert m.cache.read("drafts").tolist() == [-1] * R
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=GPU)  # noqa: E731
    count, rejected, accepted, out, drafts = i32(R), i32(R), i32(R), i32(R, D + 1), i32(D, R)
    logits, q, u = torch.zeros(ROWS, V, device=GPU), torch.zeros(D, R, V, device=GPU), torch.zeros(R, D + 1, device=GPU)
    rows = [torch.zeros(ROWS, h, HD, device=GPU) for h in (HEADS, KV, KV, HEADS)]
    qr, kr, vr, y = (x.data_ptr() for x in rows)

    def step():
        m.cache.step_dev(count.data_ptr(), drop=rejected.data_ptr(), max_count=D + 1)
        m.cache.attend_dev(0, qr, kr, vr, HD ** -0.5, y)
        ctx.verify_rows_dev(logits.data_ptr(), R, V, D, drafts.data_ptr(), q.data_ptr(), u.data_ptr(), out.data_ptr(), accepted.data_ptr(), rejected=rejected.data_ptr(), starts=a["starts"],
                            n_drafts=a["drafts"], rows=ROWS)
    torch.cuda.synchronize()
    step()
    ctx.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), stream_of(ctx)
    with torch.cuda.graph(graph, stream=stream):
        step()
    waiting, refusals, served, dropped = set(), 0, 0, 0
    for turn in range(60):
        c = [0 if rng.random() < 0.1 else int(rng.integers(1, D + 2)) for _ in range(R)]
        if turn % 6 == 5 and m.steps.lens:      # a sequence ends, its slot waits for the next turn
            s = int(np.argmax(m.steps.lens))
            rejected[s], c[s] = ALL, 0
        count.copy_(ints(c))
        logits.copy_(2 * torch.from_numpy(rng.standard_normal((ROWS, V)).astype(np.float32)))
        q.copy_(torch.softmax(2 * torch.from_numpy(rng.standard_normal((D, R, V)).astype(np.float32)), -1))
        drafts.copy_(torch.from_numpy(rng.integers(0, V, (D, R)).astype(np.int32)))
        u.copy_(torch.from_numpy(rng.random((R, D + 1)).astype(np.float32)))
        u[:, :D] *= 0.4
        new = [m.rows(ROWS, h) for h in (HEADS, KV, KV)]
        for to, x in zip(rows, new):
            to.copy_(x)
        drop, before = rejected.cpu().tolist(), list(m.steps.lens)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        m.steps.step(c, drop, D + 1)
        m.steps.check(m.cache)
        T, got = len(m.steps.seqs), [out.cpu().numpy(), accepted.cpu().numpy(), rejected.cpu().numpy()]
        for kept in (m.k[0], m.v[0]):
            for s in range(R):
                kept[s] = kept[s][:m.steps.lens[s] - m.steps.counts[s]]
        m.append(0, new[1][:T], new[2][:T])
        m.compare(rows[3][:T].cpu(), new[0][:T], 0, 0, 0, HD ** -0.5)
        n = np.array(m.steps.counts) - 1
        assert m.cache.read("drafts").tolist() == n.tolist()
        starts = np.concatenate([[0], np.cumsum(m.steps.counts)])[:R]
        check(got, logits.cpu().numpy(), starts, n, drafts.cpu().numpy(), q.cpu().numpy(), u.cpu().numpy(), np.ones(R), False, D)
        for s in range(R):
            dropped += drop[s]
            if c[s] and not m.steps.counts[s]:
                refusals += 1
                waiting.add(s)
                assert m.steps.lens[s] == max(0, before[s] - drop[s]) and (got[0][s] == -1).all() and got[1][s] == got[2][s] == 0
            elif m.steps.counts[s] and s in waiting:
                served += 1
                waiting.discard(s)
    assert refusals > 10 and served > 5 and dropped > 0
