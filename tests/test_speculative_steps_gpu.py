"""Speculative steps of several requests that follow one another without the host, in one CUDA graph: pages and places from the lengths and from what the step before rejected, a quantized
product, attention over all positions and over a window, the output matrix, verification, the next tokens.  Every operator's results are compared with the formula in 64
bits on the inputs that it had."""
import numpy as np
import pytest
import torch

from densecore_b200 import blocks as B
from kv_dev_util import GPU, Mirror, stream_of
from test_verify_rows_gpu import check

pytestmark = pytest.mark.gpu
H, HEADS, KV, HD, V, R, D = 512, 4, 2, 64, 700, 4, 3
WIDE, ROWS = (HEADS + 2 * KV) * HD, R * (D + 1)
WINDOW, KEEP = 9, 2


class Array:
    def __init__(self, owner, address, shape):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i4", "data": (address, False), "version": 3}


@pytest.mark.parametrize("drafted", ["probabilities", "certain"])
def test_steps_in_one_graph(ctx, drafted):
    rng = np.random.default_rng(12)
    m = Mirror(ctx, "f32", HEADS, KV, HD, R, 60, 20, ROWS, layers=2, seed=5)
    up = lambda n, k: ctx.upload_weight(B.GGML_TYPE_Q4_K, B.random_q4k(rng, n, k, 0.002), k, n)  # noqa: E731
    qkv, head = up(WIDE, H), up(V, H)
    embed = torch.from_numpy(rng.normal(size=(V, H)).astype(np.float32)).to(GPU)
    mix = torch.from_numpy(rng.normal(size=(HEADS * HD, H)).astype(np.float32)).to(GPU) * 0.3
    a = m.cache.arrays()
    view = {k: torch.as_tensor(Array(m.cache, a[k], s), device=GPU) for k, s in (("starts", (R + 1,)), ("seqs", (ROWS,)), ("counts", (R,)))}
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=GPU)  # noqa: E731
    n_drafts, drafts, rejected, accepted, out = i32(R), i32(D, R), i32(R), i32(R), i32(R, D + 1)
    last = torch.arange(3, 3 + R, dtype=torch.int32, device=GPU)
    q = torch.zeros(D, R, V, device=GPU)
    u, temperature = torch.zeros(R, D + 1, device=GPU), torch.tensor([0.7, 0.0, 1.0, 1.3], device=GPU)
    rows = [torch.zeros(ROWS, WIDE, device=GPU) for _ in range(2)]
    y = [torch.zeros(ROWS, HEADS * HD, device=GPU) for _ in range(2)]
    x = [torch.zeros(ROWS, H, device=GPU) for _ in range(3)]
    logits = torch.zeros(ROWS, V, device=GPU)
    q_at = q.data_ptr() if drafted == "probabilities" else 0
    place = torch.arange(ROWS, device=GPU)

    def verify():
        ctx.verify_rows_dev(logits.data_ptr(), R, V, D, drafts.data_ptr(), q_at, u.data_ptr(), out.data_ptr(), accepted.data_ptr(), rejected=rejected.data_ptr(), starts=a["starts"],
                            n_drafts=n_drafts.data_ptr(), temperature=temperature.data_ptr(), rows=ROWS)

    def step(count):
        m.cache.step_dev(count.data_ptr(), drop=rejected.data_ptr(), max_count=D + 1)
        of = view["seqs"].long().clamp(0, R - 1)
        i = (place - view["starts"].long()[of]).clamp(0, D)
        x[0].copy_(embed[torch.where(i == 0, last[of], drafts[(i - 1).clamp(min=0), of]).long()])
        for layer in range(2):
            ctx.mul_mat_dev(qkv, x[layer].data_ptr(), ROWS, rows[layer].data_ptr())
            at = rows[layer].data_ptr()
            m.cache.attend_dev(layer, at, at + 4 * HEADS * HD, at + 4 * (HEADS + KV) * HD, HD ** -0.5, y[layer].data_ptr(), window=WINDOW if layer else 0, keep_first=KEEP if layer else 0,
                               ld_q=WIDE, ld_kv=WIDE)
            x[layer + 1].copy_(x[layer] + y[layer] @ mix)
        ctx.mul_mat_dev(head, x[2].data_ptr(), ROWS, logits.data_ptr())
        verify()
        nxt = out.gather(1, accepted.long()[:, None])[:, 0]
        last.copy_(torch.where(nxt >= 0, nxt, last))

    count = i32(R)
    stream = stream_of(ctx)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):      # (a graph finds its kernels set up and its workspaces made)
        n_drafts.fill_(-1)
        step(count)
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(count)
    taken = 0
    for turn in range(24):
        n = rng.integers(-1, D + 1, R) if turn % 3 else np.full(R, D)
        if turn == 9:
            n[:] = -1
        n_drafts.copy_(torch.from_numpy(n.astype(np.int32)))
        count.copy_(n_drafts + 1)
        # drafts near to what the target gave last (its logits of some row), so that some are accepted
        z = torch.log_softmax(logits[torch.from_numpy(rng.integers(0, ROWS, (D, R))).to(GPU)] / 0.8, -1)
        q.copy_(torch.softmax(z, -1))
        drafts.copy_(torch.multinomial(q.view(-1, V), 1, generator=torch.Generator(GPU).manual_seed(turn)).view(D, R).int())
        u.copy_(torch.from_numpy(rng.random((R, D + 1)).astype(np.float32)))
        if turn % 4 == 1:
            u[:, :D] *= 0.01      # (nearly all accepted)
        drop, before = rejected.cpu().tolist(), [l for l in m.steps.lens]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        m.steps.step((n + 1).tolist(), drop, D + 1)
        m.steps.check(m.cache)
        assert m.steps.lens == [b - d + c for b, d, c in zip(before, drop, n + 1)]
        T = len(m.steps.seqs)
        for layer in range(2):
            for kept in (m.k[layer], m.v[layer]):
                for s in range(R):
                    kept[s] = kept[s][:m.steps.lens[s] - m.steps.counts[s]]
            r = rows[layer][:T].cpu()
            m.append(layer, r[:, HEADS * HD:(HEADS + KV) * HD].reshape(T, KV, HD), r[:, (HEADS + KV) * HD:].reshape(T, KV, HD))
            m.compare(y[layer][:T].cpu().view(T, HEADS, HD), r[:, :HEADS * HD].reshape(T, HEADS, HD), layer, WINDOW if layer else 0, KEEP if layer else 0, HD ** -0.5)
        starts = np.concatenate([[0], np.cumsum(n + 1)])[:R]
        check((out.cpu().numpy(), accepted.cpu().numpy(), rejected.cpu().numpy()), logits.cpu().numpy(), starts, n, drafts.cpu().numpy(), q.cpu().numpy() if q_at else None, u.cpu().numpy(),
              temperature.cpu().numpy(), False, D)
        taken += int(accepted.sum())
    assert taken > 0 and max(m.steps.lens) > 2 * WINDOW
