"""Steps of several requests as a serving program makes them: a quantized product with each request's adapter on top, attention over the cache in 4 bits on the
rows of that fused projection, the output matrix, one token a row by each request's own settings; requests join, are forked and leave.  Everything is enqueued without
waiting; each operator's results are then compared with the formula in 64 bits on the inputs that it had."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import blocks as B
from test_kv_q4_gpu import attention, held
from test_sample_rows_gpu import reference

pytestmark = pytest.mark.gpu
GPU = "cuda"
H, HEADS, KV, HD, V = 512, 4, 2, 128, 1003
WIDE = (HEADS + 2 * KV) * HD


class Engine:
    def __init__(self, ctx, rng):
        self.ctx = ctx
        self.embed = torch.from_numpy(rng.normal(size=(V, H)).astype(np.float32)).to(GPU)
        up = lambda n, k: ctx.upload_weight(B.GGML_TYPE_Q4_K, B.random_q4k(rng, n, k, 0.002), k, n)
        self.qkv, self.head = up(WIDE, H), up(V, H)
        self.cache = ctx.kv_cache_q4(1, HEADS, KV, HD, 40, 6, 12)
        self.lora = ctx.lora(H, WIDE, 3, 8)
        self.A = [torch.randn(r, H, device=GPU).mul_(H ** -0.5).bfloat16() for r in (8, 3)]
        self.B = [torch.randn(WIDE, r, device=GPU).mul_(0.2).bfloat16() for r in (8, 3)]
        torch.cuda.synchronize()
        for i, r in enumerate((8, 3)):
            self.lora.set_dev(i, r, self.A[i].data_ptr(), self.B[i].data_ptr(), 0.5 + i)
        self.keep = []

    def step(self, seqs, pos0, tokens, adapters, settings, u):
        """tokens: one list per request (a prompt or one token).  Enqueues; returns the device tensors of the step."""
        counts = [len(t) for t in tokens]
        T, n = sum(counts), len(seqs)
        x = self.embed[torch.tensor(sum(tokens, []), device=GPU)]
        ids = torch.tensor(sum(([a] * c for a, c in zip(adapters, counts)), []), dtype=torch.int32, device=GPU)
        T_, k, p, m = (torch.tensor([s[i] for s in settings], dtype=torch.int32 if i == 1 else torch.float32, device=GPU) for i in range(4))
        uu = torch.tensor(u, dtype=torch.float32, device=GPU)
        ends = torch.tensor(np.cumsum(counts) - 1, device=GPU)
        rows, plain, out = torch.empty(T, WIDE, device=GPU), torch.empty(T, WIDE, device=GPU), torch.empty(T, HEADS * HD, device=GPU)
        kh, vh = (torch.empty(T, KV, HD, device=GPU) for _ in "kv")
        logits, token, prob = torch.empty(n, V, device=GPU), torch.empty(n, dtype=torch.int32, device=GPU), torch.empty(n, device=GPU)
        torch.cuda.current_stream().synchronize()
        c = self.ctx
        self.cache.batch(seqs, pos0, counts)
        c.mul_mat_dev(self.qkv, x.data_ptr(), T, plain.data_ptr())
        c.mul_mat_lora_dev(self.qkv, self.lora, x.data_ptr(), T, ids.data_ptr(), rows.data_ptr())
        at = rows.data_ptr()
        self.cache.attend_dev(0, at, at + 4 * HEADS * HD, at + 4 * (HEADS + KV) * HD, HD ** -0.5, out.data_ptr(), ld_q=WIDE, ld_kv=WIDE, k_held=kh.data_ptr(), v_held=vh.data_ptr())
        # the last rows' results are the next product's input: on the library's stream, as a program's own kernel would be
        with torch.cuda.stream(torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(c.handle))):
            last = out[ends].contiguous()
        c.mul_mat_dev(self.head, last.data_ptr(), n, logits.data_ptr())
        c.sample_rows_dev(logits.data_ptr(), n, V, T_.data_ptr(), k.data_ptr(), p.data_ptr(), m.data_ptr(), uu.data_ptr(), token.data_ptr(), p=prob.data_ptr())
        r = dict(x=x, ids=ids, rows=rows, plain=plain, out=out, kh=kh, vh=vh, logits=logits, token=token, prob=prob, seqs=list(seqs), pos0=list(pos0), counts=counts,
                 settings=settings, u=u, more=(T_, k, p, m, uu, ends, last))
        self.keep.append(r)
        return r

    def check(self, r, K, Vv):
        """K, Vv: values that the cache stood for before the step, by sequence; brought up to date."""
        y = r["plain"].double()
        size = torch.zeros_like(y)
        for a in range(2):
            t = (r["ids"] == a).nonzero()[:, 0]
            A, Bm = self.A[a].double(), self.B[a].double()
            y[t] += (0.5 + a) * (r["x"][t].double() @ A.T @ Bm.T)
            size[t] = (0.5 + a) * (r["x"][t].double().abs() @ A.abs().T @ Bm.abs().T)
        assert torch.all((r["rows"].double() - y).abs() <= size * ((H + 8) / 8 + 24) * 2.0 ** -23 + y.abs() * 2.0 ** -24)
        rows = r["rows"].cpu().numpy()
        q = rows[:, :HEADS * HD].reshape(-1, HEADS, HD)
        k, v = (rows[:, (HEADS + i * KV) * HD:(HEADS + (i + 1) * KV) * HD].reshape(-1, KV, HD) for i in (0, 1))
        assert np.array_equal(r["kh"].cpu().numpy(), held(k)) and np.array_equal(r["vh"].cpu().numpy(), held(v))
        out, at = r["out"].cpu().numpy().reshape(-1, HEADS, HD), 0
        for s, p, n in zip(r["seqs"], r["pos0"], r["counts"]):
            K[s], Vv[s] = np.concatenate([K[s][:p], held(k[at:at + n])]), np.concatenate([Vv[s][:p], held(v[at:at + n])])
            want, tol = attention(q[at:at + n], K[s], Vv[s], p, HD ** -0.5)
            assert np.all(np.abs(out[at:at + n] - want) <= tol)
            at += n
        logits, token, prob = r["logits"].cpu().numpy(), r["token"].cpu().numpy(), r["prob"].cpu().numpy()
        for i, s in enumerate(r["settings"]):
            want, p, _, _, decided = reference(logits[i], np.float32(s[0]), s[1], np.float32(s[2]), np.float32(s[3]), np.float32(r["u"][i]))
            if decided:
                assert token[i] == want and abs(prob[i] - p) <= 2.0 ** -23 * p


def test_requests_join_fork_and_leave(ctx):
    rng = np.random.default_rng(77)
    e = Engine(ctx, rng)
    empty = np.zeros((0, KV, HD), np.float32)
    settings = {0: (0.8, 40, 0.95, 0.0), 1: (0.0, 0, 1.0, 0.0), 2: (1.2, 0, 0.9, 0.05), 3: (1.0, 0, 1.0, 0.0)}
    K, Vv, length, last, adapter = {}, {}, {}, {}, {}
    done = []

    def step(batch):
        seqs = list(batch)
        r = e.step(seqs, [length[s] for s in seqs], [batch[s] for s in seqs], [adapter[s] for s in seqs], [settings[s % 4] for s in seqs], list(rng.random(len(seqs))))
        for s, n in zip(seqs, r["counts"]):
            length[s] += n
        done.append(r)
        tokens = r["token"].cpu().numpy()      # (the program needs them for its next step)
        for s, t in zip(seqs, tokens):
            assert 0 <= t < V
            last[s] = int(t)

    def join(a):
        s = e.cache.seq_alloc()
        K[s], Vv[s], length[s], adapter[s] = empty, empty, 0, a
        return s

    def settle():
        ctx.synchronize()
        for r in done:
            e.check(r, K, Vv)
        done.clear()

    a, b = join(0), join(-1)
    ctx.synchronize()
    step({a: list(rng.integers(0, V, 37)), b: list(rng.integers(0, V, 5))})
    step({a: [last[a]], b: [last[b]]})
    c = join(1)
    step({c: list(rng.integers(0, V, 70)), a: [last[a]], b: [last[b]]})
    settle()
    f = e.cache.seq_fork(c)
    K[f], Vv[f], length[f], last[f], adapter[f] = K[c].copy(), Vv[c].copy(), length[c], last[c], 0
    for _ in range(4):
        step({s: [last[s]] for s in (f, c, a, b)})
    settle()
    free = e.cache.free_blocks()
    e.cache.seq_free(c)
    assert e.cache.free_blocks() > free
    d = join(2)                                # an adapter that is not there
    step({d: list(rng.integers(0, V, 20)), f: [last[f]], a: [last[a], 5, 6]})
    step({d: [last[d]], f: [last[f]], a: [last[a]], b: [last[b]]})
    settle()
    e.cache.close()
    e.lora.close()
    e.qkv.free()
    e.head.free()
