"""Plain restatements of a cache whose sequences are kept on the GPU, for its tests: steps in numpy, attention in 64 bits."""
import numpy as np
import torch

import densecore_b200 as dc

GPU = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int64).clip(-2**31, 2**31 - 1), dtype=torch.int32, device=GPU)


class Steps:
    """Lengths, pages, tables and the stack of free pages."""

    def __init__(self, slots, pages, a_slot, max_tokens):
        self.a_slot, self.max_tokens = a_slot, max_tokens
        self.lens, self.counts = [0] * slots, [0] * slots
        self.tables = [[] for _ in range(slots)]
        self.stack = list(range(pages - 1, -1, -1))
        self.slots, self.positions, self.seqs = [], [], []

    def step(self, count, drop, max_count):
        n = len(self.lens)
        keep = [l - min(max(d, 0), l) for l, d in zip(self.lens, drop)]
        ask = [c if 0 <= c <= max_count and k + c <= 16 * self.a_slot else 0 for c, k in zip(count, keep)]
        need = [-(-(k + c) // 16) for k, c in zip(keep, ask)]
        freed, left = [], []
        for t, m in zip(self.tables, need):
            freed += t[m:]
            left.append(t[:m])
        there, wanted, tokens, missing = len(self.stack) + len(freed), 0, 0, []
        for s in range(n):
            more = need[s] - len(left[s])
            wanted, tokens = wanted + more, tokens + ask[s]
            if (more and wanted > there) or tokens > self.max_tokens:
                ask[s] = more = 0
            missing.append(more)
        self.stack += freed[::-1]
        for s in range(n):
            left[s] = left[s] + [self.stack.pop() for _ in range(missing[s])]
        self.tables, self.counts = left, ask
        self.lens = [k + c for k, c in zip(keep, ask)]
        self.seqs = [s for s in range(n) for _ in range(ask[s])]
        self.positions = [keep[s] + i for s in range(n) for i in range(ask[s])]
        self.slots = [self.tables[s][p // 16] * 16 + p % 16 for s, p in zip(self.seqs, self.positions)]

    def check(self, kv):
        n, T = len(self.lens), len(self.seqs)
        assert kv.read("lens").tolist() == self.lens
        assert kv.read("counts").tolist() == self.counts
        assert kv.read("starts").tolist() == np.concatenate([[0], np.cumsum(self.counts)]).tolist()
        assert kv.read("free").tolist() == [len(self.stack)]
        tables = kv.read("tables")
        for s in range(n):
            assert tables[s, :len(self.tables[s])].tolist() == self.tables[s], s
        for name, want in (("slots", self.slots), ("positions", self.positions), ("seqs", self.seqs)):
            assert kv.read(name)[:T].tolist() == want, name


class Mirror:
    """A cache on the GPU beside its steps and its rows in 64 bits."""

    def __init__(self, ctx, dtype, heads, n_kv, hd, slots, pages, a_slot, max_tokens, layers=1, seed=0):
        self.ctx, self.dtype, self.heads, self.n_kv, self.hd, self.layers = ctx, dtype, heads, n_kv, hd, layers
        self.cache = ctx.kv_cache_dev(layers, heads, n_kv, hd, pages, slots, a_slot, max_tokens, dtype=dtype)
        self.steps = Steps(slots, pages, a_slot, max_tokens)
        self.k, self.v = ([[np.zeros((0, n_kv, hd)) for _ in range(slots)] for _ in range(layers)] for _ in "kv")
        self.rng = torch.Generator("cpu").manual_seed(seed)

    def step(self, count, drop=None, max_count=None):
        drop = drop or [0] * len(count)
        max_count = max(count) if max_count is None else max_count
        c, d = ints(count), ints(drop)
        torch.cuda.synchronize()
        self.cache.step_dev(c.data_ptr(), drop=d.data_ptr(), max_count=max_count)
        self.ctx.synchronize()
        self.steps.step(count, drop, max_count)
        for layer in range(self.layers):
            for rows in (self.k[layer], self.v[layer]):
                for s in range(len(count)):
                    rows[s] = rows[s][:self.steps.lens[s] - self.steps.counts[s]]

    def rows(self, n, heads, scale=1.0):
        return (scale * torch.randn(n, heads, self.hd, generator=self.rng)).to(TYPES[self.dtype])

    def held(self, x):
        return x.to(torch.float16 if self.dtype == "f32" else x.dtype).double().numpy()

    def append(self, layer, k, v):
        at = 0
        for s, n in enumerate(self.steps.counts):
            for rows, x in ((self.k[layer], k), (self.v[layer], v)):
                rows[s] = np.concatenate([rows[s], self.held(x[at:at + n])])
            at += n

    def attend(self, layer=0, window=0, keep=0, scale=None, q=None, k=None, v=None, pad=(0, 0, 0), shift=(0, 0, 0), written=False):
        """One call over the step, compared; pad: elements behind a row of q, k and v, out; shift: elements ahead of the first one of each."""
        T, t = len(self.steps.seqs), TYPES[self.dtype]
        scale = self.hd ** -0.5 if scale is None else scale
        q = self.rows(T, self.heads, 2.0) if q is None else q
        k, v = (self.rows(T, self.n_kv) if x is None else x for x in (k, v))
        room = max(T, 1) + 3

        def lay(x, heads, pad, shift):
            ld = heads * self.hd + pad
            buf = torch.full((room * ld + shift + 16,), -7.0, dtype=t)
            view = buf[shift:shift + room * ld].view(room, ld)[:, :heads * self.hd]
            if x is not None:
                view[:T] = x.reshape(T, -1)
            buf = buf.to(GPU)
            return buf, buf.data_ptr() + shift * buf.element_size(), ld
        (qb, qa, ldq), (kb, ka, ldk), (vb, va, _), (ob, oa, ldo) = lay(q, self.heads, pad[0], shift[0]), lay(k, self.n_kv, pad[1], shift[1]), lay(v, self.n_kv, pad[1], shift[1]), \
            lay(None, self.heads, pad[2], shift[2])
        torch.cuda.synchronize()
        if written:
            self.cache.write_dev(layer, ka, va, ld=ldk)
            self.cache.attend_dev(layer, qa, 0, 0, scale, oa, window=window, keep_first=keep, ld_q=ldq, ld_out=ldo)
        else:
            self.cache.attend_dev(layer, qa, ka, va, scale, oa, window=window, keep_first=keep, ld_q=ldq, ld_kv=ldk, ld_out=ldo)
        self.ctx.synchronize()
        self.append(layer, k, v)
        got = ob.cpu()
        rows = got[shift[2]:shift[2] + room * ldo].view(room, ldo)
        assert (rows[T:] == -7).all() and (rows[:, self.heads * self.hd:] == -7).all() and (got[:shift[2]] == -7).all()
        out = rows[:T, :self.heads * self.hd].reshape(T, self.heads, self.hd)
        self.compare(out, q, layer, window, keep, scale)
        return out

    def compare(self, out, q, layer, window, keep, scale):
        """Row by row against 64 bits.  What a result may be off by, of the weighted sum A of its values' sizes: twice the relative error of a weight, and of f32 sums over as many
        steps of sixteen keys.  A weight's: that of its score (queries in two fp16 terms, 2^-22 of the row's largest, where rows are f32; f32 sums of HD products, 2^-21 of their sizes), of exp2
        (2^-21) and of its two terms (fp16 2^-22, bf16 2^-18).  Then its own rounding.
        Sequences of more than 64 rows of 16 bits have weights of one term (fp16 2^-12, bf16 2^-9), whose sum is that of the rounded ones: weights w (1 + d) with |d| <= 2^-9 give
        sum w (1 + d) (v - y) / sum w (1 + d) off y, which is at most 2^-9 (A + |y|) and 2^-18 of that, so twice 2^-9 of A as |y| <= A."""
        out, q = out.double().numpy(), q.double().numpy()
        eps = torch.finfo(TYPES[self.dtype]).eps / 2
        G, t = self.heads // self.n_kv, 0
        for s, n in enumerate(self.steps.counts):
            K, V = self.k[layer][s], self.v[layer][s]
            one = n * G > 64
            terms = {"f32": 2.0**-20, "f16": 2.0**-11.99 if one else 2.0**-20, "bf16": 2.0**-8.99 if one else 2.0**-17}[self.dtype]
            for p in range(self.steps.lens[s] - n, self.steps.lens[s]):
                at = np.arange(p + 1)
                at = at[(at > p - window) | (at < keep)] if window else at
                for h in range(self.n_kv):
                    ks, vs = K[at, h], V[at, h]
                    qs = q[t, h * G:(h + 1) * G]
                    with np.errstate(all="ignore"):
                        z = qs @ ks.T * scale
                        w = np.exp(z - z.max(1, keepdims=True))
                        w /= w.sum(1, keepdims=True)
                        y = w @ vs
                        sizes = abs(scale) * np.max(np.abs(qs) @ np.abs(ks).T, 1, keepdims=True)
                        score = sizes * 2.0**-21
                        if self.dtype == "f32":
                            score = score + abs(scale) * np.abs(qs).max(1, keepdims=True) * np.abs(ks).sum(1).max() * 2.0**-22
                        A = w @ np.abs(vs)
                        bound = (2 * (score + terms) + (len(at) / 16 + 8) * 2.0**-23) * A + (eps + 2.0**-24) * np.abs(y) + 1e-30
                        if self.dtype == "f16":
                            bound = bound + 2.0**-25
                    got = out[t, h * G:(h + 1) * G]
                    # (a weight is two terms, of which the second may be 0 or less: an infinite value times their sum is infinity, times each of them NaN)
                    assert np.array_equal(np.isfinite(got), np.isfinite(y)) and np.isnan(got[np.isnan(y)]).all(), (s, p, h)
                    fine = np.isfinite(y)
                    worst = np.max(np.where(fine, np.abs(got - y) / bound, 0.0), initial=0.0)
                    assert worst <= 1.0, (s, p, h, worst)
                t += 1


def stream_of(ctx):
    return torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
