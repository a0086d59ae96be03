"""Verification of many requests' drafted tokens against 64 bits.  A decision that hangs on less than the stated accuracy of weights may go either way."""
import numpy as np
import pytest
import torch

import densecore_b200 as dc
from kv_dev_util import GPU, stream_of

pytestmark = pytest.mark.gpu
# weights are exact to 2^-22 and a row's sum of them to as much: a share of them to 2^-20, with room for the rounding of shares that are subtracted
CLOSE = 2.0**-20


def target_of(x, T, probs):
    x = x.astype(np.float64)
    if probs:
        return np.where((x > 0) & np.isfinite(x), x, 0.0)
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return np.zeros_like(x)
    if not T > 0:
        p = np.zeros_like(x)
        p[int(x.argmax())] = 1.0
        return p
    if x.max() == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.exp((x - x.max()) / T)
    return w / w.sum()


def check(got, target, starts, n_drafts, tokens, q, u, T, probs, D):
    """got: (tokens [R][D + 1], accepted, rejected)."""
    V = target.shape[1]
    for r in range(len(starts)):
        n = min(n_drafts[r], D)
        if n < 0 or starts[r] < 0 or starts[r] + n >= len(target):
            assert got[0][r].tolist() == [-1] * (D + 1) and got[1][r] == 0 and got[2][r] == 0, r
            continue
        k = got[1][r]
        assert 0 <= k <= n and got[2][r] == n - k and got[0][r, :k].tolist() == [tokens[i][r] for i in range(k)] and (got[0][r, k + 1:] == -1).all(), r
        for i in range(min(k + 1, n)):
            t = tokens[i][r]
            p = target_of(target[starts[r] + i], T[r], probs)
            good = 0 <= t < V
            if good:
                qt = 1.0 if q is None else float(q[i, r, t]) if q[i, r, t] > 0 and np.isfinite(q[i, r, t]) else 0.0
                uq = float(u[r, i]) * qt
                if abs(uq - p[t]) <= CLOSE * p[t] and p[t] > 0:
                    continue
                good = uq < p[t]
            assert good == (i < k), (r, i)
        p = target_of(target[starts[r] + k], T[r], probs)
        w = p
        if k < n:
            if q is None:
                qr = np.zeros(V)
                if 0 <= tokens[k][r] < V:
                    qr[tokens[k][r]] = 1.0
            else:
                qr = np.where((q[k, r] > 0) & np.isfinite(q[k, r]), q[k, r].astype(np.float64), 0.0)
            w = np.maximum(p - qr, 0.0)
            if w.sum() <= CLOSE * p.sum():      # nothing but rounding: either from it or from p
                continue
        if w.sum() == 0:
            assert got[0][r, k] == -1, r
            continue
        upto = np.cumsum(w)
        t, off = got[0][r, k], CLOSE * p.sum()
        goal = float(u[r, D]) * upto[-1]
        assert 0 <= t < V and w[t] > -off and (t == 0 or upto[t - 1] <= goal + off) and upto[t] > goal - off and p[t] > 0, (r, k, t)


def run(ctx, target, starts, n_drafts, tokens, q, u, T, probs=False, dtype="f32", ld=0, shift=0):
    R, D = len(n_drafts), u.shape[1] - 1
    V = target.shape[1]
    ld = ld or V
    buf = torch.full((shift + len(target) * ld,), 7.0, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32)
    buf[shift:].view(len(target), ld)[:, :V] = torch.from_numpy(target)
    buf = buf.to(GPU)
    put = lambda a, t: None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype=t)).to(GPU)  # noqa: E731
    s, n, tk, qd, ud, Td = put(starts, np.int32), put(n_drafts, np.int32), put(tokens if D else np.zeros((1, R)), np.int32), put(q, np.float32), put(u, np.float32), put(T, np.float32)
    out, acc, rej = torch.full((R, D + 1), -9, dtype=torch.int32, device=GPU), torch.full((R,), -9, dtype=torch.int32, device=GPU), torch.full((R,), -9, dtype=torch.int32, device=GPU)
    torch.cuda.synchronize()
    ctx.verify_rows_dev(buf.data_ptr() + shift * buf.element_size(), R, V, D, tk.data_ptr(), qd.data_ptr() if qd is not None else 0, ud.data_ptr(), out.data_ptr(), acc.data_ptr(),
                        rejected=rej.data_ptr(), starts=s.data_ptr(), n_drafts=n.data_ptr(), temperature=Td.data_ptr() if not probs else 0, rows=len(target), ld=ld, dtype=dtype, probs=probs)
    ctx.synchronize()
    got = out.cpu().numpy(), acc.cpu().numpy(), rej.cpu().numpy()
    seen = buf[shift:].view(len(target), ld)[:, :V].float().cpu().numpy()
    check(got, seen, starts, n_drafts, tokens, q, u, T if T is not None else np.ones(R), probs, D)
    return got


def make(rng, R, D, V, near=0.5, probs=False, steep=3.0):
    """Rows that fall steeply, drafts from distributions near them, requests of all numbers of drafts, one in eight without part."""
    n = rng.integers(0, D + 1, R)
    n[rng.random(R) < 0.4] = D
    n[rng.random(R) < 0.12] = -1
    starts = np.concatenate([[0], np.cumsum(np.maximum(n, -1) + 1)[:-1]])
    x = (steep * rng.standard_normal((int((n + 1).sum()) + 1, V))).astype(np.float32)
    T = rng.choice([0.0, 0.6, 1.0, 1.4], R).astype(np.float32)
    q = np.zeros((D, R, V), np.float32)
    tokens = np.zeros((D, R), np.int32)
    for i in range(D):
        for r in range(R):
            y = x[min(starts[r] + i, len(x) - 1)] + near * rng.standard_normal(V)
            q[i, r] = target_of(y, T[r], False)
            tokens[i, r] = min(V - 1, int((np.cumsum(q[i, r].astype(np.float64)) <= rng.random()).sum()))
    if probs:
        x = np.stack([target_of(r, 1.0, False) for r in x]).astype(np.float32)
    return x, starts, n, tokens, q, rng.random((R, D + 1)).astype(np.float32), T


@pytest.mark.parametrize("form", ["f32", "bf16", "probs"])
@pytest.mark.parametrize("R,D,V", [(1, 0, 5), (1, 1, 1), (3, 2, 2), (9, 4, 7), (40, 3, 90), (5, 8, 2047), (6, 4, 2048), (4, 5, 2049), (30, 2, 5000), (2, 4, 32001), (3, 3, 151936), (700, 1, 257), (2, 64, 300)])
def test_requests_against_64_bits(ctx, form, R, D, V):
    rng = np.random.default_rng(R * 1000 + V)
    x, starts, n, tokens, q, u, T = make(rng, R, D, V, probs=form == "probs")
    got = run(ctx, x, starts, n, tokens, q, u, T, probs=form == "probs", dtype="bf16" if form == "bf16" else "f32")
    if R * D > 50:
        assert 0 < got[1].sum() < np.maximum(n, 0).sum()
    run(ctx, x, starts, n, tokens, None, u, T, probs=form == "probs", dtype="bf16" if form == "bf16" else "f32")


@pytest.mark.parametrize("form", ["f32", "bf16", "probs"])
def test_requests_that_share_rows(ctx, form):
    """Several requests' rows may be the same ones, wholly or in part, and in any order."""
    rng = np.random.default_rng(21)
    D, V = 3, 2500
    x, _, _, tokens, q, u, T = make(rng, 8, D, V, probs=form == "probs")
    x, starts, n = x[:5], np.array([0, 0, 1, 1, 0, 1, 4, 0]), np.array([3, 3, 3, 2, 0, 3, 0, 1])
    run(ctx, x, starts, n, tokens, q, u, T, probs=form == "probs", dtype="bf16" if form == "bf16" else "f32")


@pytest.mark.parametrize("dtype,ld,shift", [("f32", 0, 1), ("f32", 3001, 0), ("f32", 3004, 4), ("bf16", 0, 3), ("bf16", 3007, 0), ("bf16", 3008, 8), ("probs", 3003, 2)])
def test_rows_of_any_alignment(ctx, dtype, ld, shift):
    rng = np.random.default_rng(5)
    x, starts, n, tokens, q, u, T = make(rng, 12, 3, 3000, probs=dtype == "probs")
    run(ctx, x, starts, n, tokens, q, u, T, probs=dtype == "probs", dtype="f32" if dtype == "probs" else dtype, ld=ld, shift=shift)


def test_draws_follow_the_uniform_number(ctx):
    """One row, uniform numbers from 0 to just below 1: tokens rise, and each comes as often as its share says."""
    V, R = 300, 4000
    rng = np.random.default_rng(2)
    x = np.repeat((2 * rng.standard_normal((1, V))).astype(np.float32), R, 0)
    u = np.linspace(0, 1, R, endpoint=False, dtype=np.float32)[:, None]
    u[-1] = np.nextafter(np.float32(1), np.float32(0))
    got = run(ctx, x, np.arange(R), np.zeros(R, int), np.zeros((0, R)), np.zeros((0, R, V)), u, np.ones(R, np.float32))
    t = got[0][:, 0]
    assert (np.diff(t) >= 0).all()
    assert np.abs(np.bincount(t, minlength=V) / R - target_of(x[0], 1.0, False)).max() <= 1.5 / R


def test_masked_and_infinite_logits(ctx):
    """Rows with -inf, NaN, +inf, the type's lowest value, one token left, and none: no weight, all weight, or token -1."""
    V = 2500
    rng = np.random.default_rng(3)
    low = np.finfo(np.float32).min
    rows = []
    for fill in ("some", "one", "none", "nan", "inf", "twoinf", "low", "alllow", "far"):
        for _ in range(2):
            x = (3 * rng.standard_normal(V)).astype(np.float32)
            if fill == "some":
                x[rng.random(V) < 0.7] = -np.inf
            elif fill == "one":
                x[:] = -np.inf
                x[2100] = 1.0
            elif fill == "none":
                x[:] = -np.inf
            elif fill == "nan":
                x[rng.random(V) < 0.5] = np.nan
            elif fill == "inf":
                x[77] = np.inf
            elif fill == "twoinf":
                x[[5, 2400]] = np.inf
            elif fill == "low":
                x[rng.random(V) < 0.5] = low
            elif fill == "alllow":
                x[:] = low
            elif fill == "far":
                x[::2] -= 200.0
            rows.append(x)
    R = len(rows) // 2
    x = np.stack(rows)
    q = np.stack([np.stack([target_of((2 * rng.standard_normal(V)), 1.0, False) for _ in range(R)])]).astype(np.float32)
    tokens = np.array([[2100, 5, 77, 0, 77, 5, 9, 3, 1]], np.int32)
    for T in (0.0, 1e-38, 0.5, 1.0, 1e6):
        for _ in range(4):
            run(ctx, x, 2 * np.arange(R), np.ones(R, int), tokens, q, rng.random((R, 2)).astype(np.float32), np.full(R, T, np.float32))


def test_drafts_that_are_nowhere_below_the_target(ctx):
    """A draft as probable as the target says is accepted; one with twice the target's probabilities is rejected at a high number, and the next token then comes from the target."""
    V, R = 700, 64
    rng = np.random.default_rng(4)
    p = rng.random((2 * R, V)).astype(np.float32)
    p /= p.sum(1, keepdims=True)
    q = p[0::2][None]
    tokens = rng.integers(0, V, (1, R)).astype(np.int32)
    u = (0.9 * rng.random((R, 2))).astype(np.float32)
    got = run(ctx, p, 2 * np.arange(R), np.ones(R, int), tokens, q, u, None, probs=True)
    assert (got[1] == 1).all()
    u[:, 0] = 0.75
    got = run(ctx, p, 2 * np.arange(R), np.ones(R, int), tokens, 2 * q, u, None, probs=True)
    assert (got[1] == 0).all()
    for r in range(R):      # nothing is left of p - 2 p
        upto = np.cumsum(p[2 * r].astype(np.float64))
        t = got[0][r, 0]
        assert (t == 0 or upto[t - 1] <= u[r, 1] * upto[-1] * (1 + CLOSE)) and upto[t] >= u[r, 1] * upto[-1] * (1 - CLOSE)


def test_bad_device_numbers_are_harmless(ctx):
    """Tokens outside the vocabulary are rejected; probabilities that are negative, NaN or infinite count as none; rows outside the target's leave a request out."""
    V, R, D = 400, 8, 2
    rng = np.random.default_rng(6)
    x = (2 * rng.standard_normal((R * 3, V))).astype(np.float32)
    tokens = rng.integers(0, V, (D, R)).astype(np.int32)
    tokens[0, :4] = [-1, V, 2**31 - 1, -2**31]
    q = np.abs(rng.standard_normal((D, R, V))).astype(np.float32) / V
    q[:, :, ::5], q[:, :, 1::7], q[:, :, 2::11] = np.nan, -1.0, np.inf
    starts = 3 * np.arange(R)
    starts[4:7] = [-1, 22, 2**31 - 1]
    n = np.array([2, 2, 1, 2, 2, 2, 0, 99])
    run(ctx, x, starts, n, tokens, q, rng.random((R, D + 1)).astype(np.float32), np.ones(R, np.float32))


def test_host_arrays(ctx):
    rng = np.random.default_rng(7)
    R, D, V = 6, 3, 1000
    x = (2 * rng.standard_normal((R, D + 1, V))).astype(np.float32)
    q = np.stack([np.stack([target_of(x[r, i] + 0.4 * rng.standard_normal(V), 1.0, False) for r in range(R)]) for i in range(D)]).astype(np.float32)
    tokens = q.argmax(2).astype(np.int32)
    u = rng.random((R, D + 1)).astype(np.float32)
    n = np.array([3, 2, 0, 3, 1, 3])
    t, a = ctx.verify_rows(x, tokens, q, u, n_drafts=n, temperature=0.8)
    check((t, a, n - a), x.reshape(-1, V), (D + 1) * np.arange(R), n, tokens, q, u, np.full(R, 0.8), False, D)
    t2, a2 = ctx.verify_rows(x, tokens, None, u)
    check((t2, a2, D - a2), x.reshape(-1, V), (D + 1) * np.arange(R), [D] * R, tokens, None, u, np.ones(R), False, D)
    for bad in (dict(uniforms=u + 1), dict(temperature=-1.0), dict(n_drafts=n + 1), dict(uniforms=np.full_like(u, np.nan))):
        with pytest.raises(dc.DcError):
            ctx.verify_rows(**{**dict(target=x, draft_tokens=tokens, draft_probs=q, uniforms=u), **bad})
    with pytest.raises(ValueError):
        ctx.verify_rows(x, tokens[:2], q, u)


def test_agrees_with_the_rule_for_one_request(ctx):
    """dc_b200_verify_accept on the same numbers (its sums are f32: a decision within its accuracy may differ, the seeds below have none)."""
    rng = np.random.default_rng(8)
    for mode_T in (0.7, 1.0):
        for _ in range(6):
            D, V = 4, 3000
            x, starts, n, tokens, q, u, _ = make(rng, 1, D, V)
            x = np.concatenate([x] * 5)[:D + 1]
            q = np.stack([target_of(x[i] + 0.5 * rng.standard_normal(V), mode_T, False) for i in range(D)]).astype(np.float32)
            tokens = q.argmax(1).astype(np.int32)
            want = ctx.verify_accept(x, tokens, q, u[0], mode=1, temperature=mode_T)
            t, a = ctx.verify_rows(x[None], tokens[:, None], q[:, None], u, temperature=mode_T)
            assert (int(a[0]), int(t[0, a[0]])) == want


def test_captured_and_repeated(ctx):
    """A replayed graph gives what calls give, the same every time; two graphs share the workspace."""
    rng = np.random.default_rng(9)
    made = [make(rng, R, D, V) for R, D, V in ((5, 3, 20001), (64, 2, 4000))]
    graphs, stream = [], stream_of(ctx)
    for x, starts, n, tokens, q, u, T in made:
        a = [torch.from_numpy(np.ascontiguousarray(z, dtype=t)).to(GPU) for z, t in ((x, np.float32), (starts, np.int32), (n, np.int32), (tokens, np.int32), (q, np.float32), (u, np.float32), (T, np.float32))]
        R, D, V = len(n), len(tokens), x.shape[1]
        out, acc, rej = torch.empty(R, D + 1, dtype=torch.int32, device=GPU), torch.empty(R, dtype=torch.int32, device=GPU), torch.empty(R, dtype=torch.int32, device=GPU)

        def call():
            ctx.verify_rows_dev(a[0].data_ptr(), R, V, D, a[3].data_ptr(), a[4].data_ptr(), a[5].data_ptr(), out.data_ptr(), acc.data_ptr(), rejected=rej.data_ptr(), starts=a[1].data_ptr(),
                                n_drafts=a[2].data_ptr(), temperature=a[6].data_ptr(), rows=len(x))
        torch.cuda.synchronize()
        call()
        ctx.synchronize()
        want = out.clone(), acc.clone(), rej.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
        graphs.append((g, (out, acc, rej), want, a))
    for _ in range(5):
        for g, got, want, _ in graphs:
            for z in got:
                z.fill_(-5)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g, *_ in graphs:
                g.replay()
        ctx.synchronize()
        for _, got, want, _ in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
