"""Adapters of many requests beside a product, against the formula in 64 bits.

Rounding that the bounds count: rows enter the products as two terms of 11 bits (2^-22 of each number at most), sums in f32 over the length n round by at most
(n / 8 + 8) 2^-23 of the sum of the magnitudes (eight products a step), the row between the products once more (2^-24 for the scale): of S = s sum_r (sum_k |x A|) |B|
that is at most ((K + R) / 8 + 24) 2^-23 in all, plus the result's own 2^-24."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import blocks as Bk

pytestmark = pytest.mark.gpu
GPU = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Adapters:
    def __init__(self, ctx, K, N, ranks, dtype, seed=0, slots=None, max_rank=None):
        g = torch.Generator(GPU).manual_seed(seed)
        t = TYPES[dtype]
        self.ctx, self.K, self.N = ctx, K, N
        self.set = ctx.lora(K, N, slots or len(ranks), max_rank or max(ranks), dtype=dtype)
        self.A = [(torch.randn(r, K, generator=g, device=GPU) * K ** -0.5).to(t) for r in ranks]
        self.B = [(0.3 * torch.randn(N, r, generator=g, device=GPU)).to(t) for r in ranks]
        self.s = [0.25 + 0.5 * i for i in range(len(ranks))]
        torch.cuda.synchronize()
        for i, r in enumerate(ranks):
            self.set.set_dev(i, r, self.A[i].data_ptr(), self.B[i].data_ptr(), self.s[i])
        ctx.synchronize()

    def expected(self, x, base, ids):
        y, size = base.double(), torch.zeros_like(base, dtype=torch.float64)
        for a in set(ids.tolist()):
            if 0 <= a < len(self.A):
                t = (ids == a).nonzero()[:, 0]
                A, B = self.A[a].double(), self.B[a].double()
                y[t] += self.s[a] * (x[t].double() @ A.T @ B.T)
                size[t] = self.s[a] * (x[t].double().abs() @ A.abs().T @ B.abs().T)
        R = max(a.shape[0] for a in self.A)
        tol = size * ((self.K + R) / 8 + 24) * 2.0 ** -23 + y.abs() * 2.0 ** -24
        return y, tol

    def run(self, x, base, ids, in_place=False):
        y = base.clone() if in_place else torch.full_like(base, 77.0)
        torch.cuda.synchronize()
        self.ctx.lora_add_dev(self.set, x.data_ptr(), x.shape[0], ids.data_ptr(), y.data_ptr(), base_dev=0 if in_place else base.data_ptr())
        self.ctx.synchronize()
        return y

    def check(self, x, base, ids, **kw):
        y, tol = self.expected(x, base, ids)
        got = self.run(x, base, ids, **kw)
        worst = ((got.double() - y).abs() / tol.clamp(min=1e-300)).max().item() if got.numel() else 0.0
        assert worst <= 1.0, worst
        none = (ids < 0) | (ids >= len(self.A))
        assert torch.equal(got[none], base[none])


def rows(M, K, N, n, seed, order="any"):
    g = torch.Generator(GPU).manual_seed(seed)
    x, base = torch.randn(M, K, generator=g, device=GPU), torch.randn(M, N, generator=g, device=GPU)
    ids = (torch.randint(0, n + 1, (M,), generator=g, device=GPU) - 1).int()
    if order == "runs":
        ids = ids[torch.arange(M, device=GPU) // 37 * 37].contiguous()
    return x, base, ids


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("K,N", [(1, 1), (64, 60), (100, 333), (2048, 1024), (1000, 129)])
@pytest.mark.parametrize("M", [1, 2, 15, 17, 64, 128, 129, 200, 531])
def test_shapes(ctx, dtype, K, N, M):
    a = Adapters(ctx, K, N, [16, 1, 40, 7, 64], dtype, seed=K + N)
    for order in ("any", "runs"):
        a.check(*rows(M, K, N, 5, M, order))


@pytest.mark.parametrize("rank", [16, 32, 48])
@pytest.mark.parametrize("M", [96, 97, 127, 128, 255, 256, 257])
def test_where_tiles_begin(ctx, rank, M):
    a = Adapters(ctx, 320, 264, [rank, 1, rank // 2], "f16", seed=M)
    for order in ("any", "runs"):
        a.check(*rows(M, 320, 264, 3, M, order))


@pytest.mark.parametrize("M", [5, 300])
@pytest.mark.parametrize("rank", [1, 15, 16, 17, 65, 128, 200])
def test_ranks(ctx, rank, M):
    a = Adapters(ctx, 256, 200, [rank, max(1, rank // 2)], "bf16", seed=rank)
    a.check(*rows(M, 256, 200, 2, rank))


@pytest.mark.parametrize("M", [3, 150])
def test_in_place_none_unknown_and_empty(ctx, M):
    a = Adapters(ctx, 128, 96, [8, 24], "bf16", slots=5)
    x, base, ids = rows(M, 128, 96, 2, 1)
    a.check(x, base, ids, in_place=True)
    for v in (-1, -2 ** 31, 2, 4, 5, 2 ** 31 - 1):                   # none, empty slots, beyond the set
        a.check(x, base, torch.full_like(ids, v))
    a.set.clear(1)
    got = a.run(x, base, ids)
    assert torch.equal(got[ids != 0], base[ids != 0])
    a.set.set_dev(1, 24, a.A[1].data_ptr(), a.B[1].data_ptr(), a.s[1])
    ctx.synchronize()
    a.check(x, base, ids)
    # a slot taken over by an adapter of a smaller rank
    a.A[1], a.B[1] = a.A[1][:5].contiguous(), a.B[1][:, :5].contiguous()
    torch.cuda.synchronize()
    a.set.set_dev(1, 5, a.A[1].data_ptr(), a.B[1].data_ptr(), a.s[1])
    ctx.synchronize()
    a.check(x, base, ids)


@pytest.mark.parametrize("M", [9, 140])
def test_a_broken_adapter_or_row_stays_alone(ctx, M):
    """Infinite and NaN matrices and rows reach the rows that name them and no others, in one tile."""
    a = Adapters(ctx, 64, 72, [8, 8, 8], "bf16")
    a.A[1][3, 5] = float("nan")
    a.B[1][:, 2] = float("inf")
    torch.cuda.synchronize()
    a.set.set_dev(1, 8, a.A[1].data_ptr(), a.B[1].data_ptr(), 1.0)
    x, base, ids = rows(M, 64, 72, 3, 2)
    x[4] = float("nan")
    ids[4] = 2
    got = a.run(x, base, ids)
    bad = (ids == 1)
    bad[4] = True
    y, tol = a.expected(x, base, torch.where(bad, -1, ids))
    good = ~bad
    assert torch.all((got.double() - y).abs()[good] <= tol[good].clamp(min=1e-300)) and torch.isnan(got[4]).all() and not torch.isfinite(got[ids == 1]).any()


@pytest.mark.parametrize("M", [6, 135])
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_rows(ctx, M, offset):
    K, N = 96, 50
    a = Adapters(ctx, K, N, [12, 20], "f16")
    x, base, ids = rows(M, K, N, 2, 3)
    wide = [torch.full((M * (n + 5) + offset,), 4.0, device=GPU) for n in (K, N, N)]
    v = [w[offset:].view(M, n + 5)[:, :n] for w, n in zip(wide, (K, N, N))]
    v[0].copy_(x), v[1].copy_(base)
    torch.cuda.synchronize()
    ctx.lora_add_dev(a.set, v[0].data_ptr(), M, ids.data_ptr(), v[2].data_ptr(), base_dev=v[1].data_ptr(), ld_x=K + 5, ld_base=N + 5, ld_y=N + 5)
    ctx.synchronize()
    y, tol = a.expected(x, base, ids)
    assert torch.all((v[2].double() - y).abs() <= tol.clamp(min=1e-300))
    rest = wide[2].clone()
    rest[offset:].view(M, N + 5)[:, :N] = 4.0
    assert torch.all(rest == 4.0)


def test_host_matrices_and_the_product_beside(ctx):
    rng = np.random.default_rng(4)
    K, N = 512, 300
    W = ctx.upload_weight(Bk.GGML_TYPE_Q4_K, Bk.random_q4k(rng, N, K), K, N)
    a = Adapters(ctx, K, N, [16, 4], "bf16")
    other = ctx.lora(K, N, 2, 16)
    for i in range(2):
        other.set(i, a.A[i].view(torch.uint16).cpu().numpy(), a.B[i].view(torch.uint16).cpu().numpy(), a.s[i])
    for M in (1, 7, 40, 200):
        x, _, ids = rows(M, K, N, 2, M)
        y, both, plain = (torch.zeros(M, N, device=GPU) for _ in range(3))
        torch.cuda.synchronize()
        ctx.mul_mat_dev(W, x.data_ptr(), M, plain.data_ptr())
        ctx.lora_add_dev(a.set, x.data_ptr(), M, ids.data_ptr(), y.data_ptr(), base_dev=plain.data_ptr())
        ctx.mul_mat_lora_dev(W, other, x.data_ptr(), M, ids.data_ptr(), both.data_ptr())
        ctx.synchronize()
        assert torch.equal(y, both)
        want, tol = a.expected(x, plain, ids)
        assert torch.all((y.double() - want).abs() <= tol.clamp(min=1e-300))
    W.free()


def test_calls_in_flight_with_growing_rows_and_two_sets(ctx):
    sets = [Adapters(ctx, 256, 128, [16, 8], "bf16", seed=i) for i in range(2)]
    keep = []
    for M in (1, 200, 3, 900, 64, 1500, 2):
        for a in sets:
            x, base, ids = rows(M, 256, 128, 2, M)
            y = torch.empty_like(base)
            torch.cuda.current_stream().synchronize()
            ctx.lora_add_dev(a.set, x.data_ptr(), M, ids.data_ptr(), y.data_ptr(), base_dev=base.data_ptr())
            keep.append((a, x, base, ids, y))
    ctx.synchronize()
    for a, x, base, ids, y in keep:
        want, tol = a.expected(x, base, ids)
        assert torch.all((y.double() - want).abs() <= tol.clamp(min=1e-300))


def test_captured_and_replayed(ctx):
    a = Adapters(ctx, 256, 128, [16, 8], "bf16")
    x, base, ids = rows(20, 256, 128, 2, 1)
    y = torch.empty_like(base)
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    a.check(x, base, ids)
    many = [t.contiguous() for t in rows(5000, 256, 128, 2, 2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ctx.lora_add_dev(a.set, x.data_ptr(), 20, ids.data_ptr(), y.data_ptr(), base_dev=base.data_ptr())
        with pytest.raises(dc.DcError) as e:
            ctx.lora_add_dev(a.set, many[0].data_ptr(), 5000, many[2].data_ptr(), many[1].data_ptr())
        assert e.value.status == -7
    a.check(*many)                              # the workspace grows; the captured call keeps the one it names
    for seed in (5, 6):
        for to, new in zip((x, base, ids), rows(20, 256, 128, 2, seed)):
            to.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        want, tol = a.expected(x, base, ids)
        assert torch.all((y.double() - want).abs() <= tol.clamp(min=1e-300))
    del graph


def test_refusals(ctx):
    for bad, status in ((dict(K=0), -1), (dict(N=0), -1), (dict(max_adapters=0), -1), (dict(max_rank=0), -1), (dict(max_rank=5000), -1), (dict(dtype="f32"), -7)):
        with pytest.raises(dc.DcError) as e:
            ctx.lora(**(dict(K=64, N=64, max_adapters=2, max_rank=8) | bad))
        assert e.value.status == status
    l = ctx.lora(64, 32, 2, 8)
    bits = lambda *s: np.zeros(s, np.uint16)
    for slot, A, B in ((2, bits(8, 64), bits(32, 8)), (-1, bits(8, 64), bits(32, 8)), (0, bits(9, 64), bits(32, 9))):
        with pytest.raises(dc.DcError):
            l.set(slot, A, B)
    for A, B in ((bits(8, 63), bits(32, 8)), (bits(8, 64), bits(32, 7)), (np.zeros((8, 64), np.float32), bits(32, 8))):
        with pytest.raises(ValueError):
            l.set(0, A, B)
    with pytest.raises(dc.DcError):
        l.set(0, bits(8, 64), bits(32, 8), float("inf"))
    with pytest.raises(dc.DcError):
        l.set_dev(0, 4, 0, 256)
    x = 256
    for args, kw in (((x, -1, x, x), {}), ((0, 1, x, x), {}), ((x, 1, 0, x), {}), ((x, 1, x, 0), {}), ((x, 1, x, x), dict(ld_x=63)), ((x, 1, x, x), dict(ld_y=31)), ((x, 1, x, x), dict(ld_base=31))):
        with pytest.raises(dc.DcError) as e:
            ctx.lora_add_dev(l, *args, **kw)
        assert e.value.status == -1
    ctx.lora_add_dev(l, 0, 0, 0, 0)                                  # no rows
    rng = np.random.default_rng(0)
    W = ctx.upload_weight(Bk.GGML_TYPE_Q4_K, Bk.random_q4k(rng, 32, 256), 256, 32)
    with pytest.raises(dc.DcError):
        ctx.mul_mat_lora_dev(W, l, x, 1, x, x)                        # another shape
    l2 = ctx.lora(256, 32, 2, 8)
    buf = torch.zeros(4096, device=GPU)
    with pytest.raises(dc.DcError):
        ctx.mul_mat_lora_dev(W, l2, buf.data_ptr(), 1, x, buf.data_ptr() + 64)      # x and y overlap
    with pytest.raises(dc.DcError):
        ctx.mul_mat_lora_dev(W, l2, buf.data_ptr(), 0, x, buf.data_ptr() + 8192)
    W.free()
