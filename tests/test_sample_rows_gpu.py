"""Sampling of many rows by temperature, top-k, top-p and min-p against the definition in 64 bits.

Tokens have to be equal.  Weights are whole numbers of 2^-44 of the largest, each off by half of one at most, so that a sum of 2^19 is off by 2^-26; sums here are
taken in 80 bits.  A row is left out of the comparison where a border between tokens, or a filter's, lies within 2^-25 of what decides; few may be.  A
row of equal values leaves none out: its sums are whole numbers on both sides.  A probability is a quotient of two such sums, rounded to f32."""
import ctypes as C

import numpy as np
import pytest
import torch

import densecore_b200 as dc

pytestmark = pytest.mark.gpu
GPU = "cuda"
NEAR = 2.0 ** -25
# Probabilities of a distribution: exp2 in f32 (2^-22), the share of one weight (2^-24), two products (2^-23), the argument (half a step of 1/2, 2^-25 ln 2): 2^-21.3 in all.
DIST = 2.0 ** -21


def reference(x, T, k, top_p, min_p, u, near=NEAR):
    """(token, probability, kept indexes by rising index, their probabilities, decided) of one row."""
    V = len(x)
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not np.any(x > -np.inf):
        return -1, 0.0, np.zeros(0, int), np.zeros(0), True
    order = np.lexsort((np.arange(V), -x))
    if not T > 0:
        return order[0], 1.0, order[:1], np.ones(1), True
    n = min(k, V) if k > 0 else V
    with np.errstate(invalid="ignore", over="ignore"):
        z = (x[order] - x[order[0]]) / np.float64(np.float32(T))
    z[x[order] == x[order[0]]] = 0.0
    z[x[order] == -np.inf] = -np.inf
    w = np.exp(z)[:n]
    decided = True
    p32, m32 = float(np.float32(top_p)), float(np.float32(min_p))
    if p32 < 1:
        ahead = np.cumsum(w, dtype=np.longdouble) - w
        goal = p32 * w.sum(dtype=np.longdouble)
        keep = max(1, int((ahead < goal).sum()))
        decided &= bool(np.abs(ahead - goal).min() > near)
        w = w[:keep]
    decided &= bool(np.all(np.abs(w - m32) > near) or m32 in (0.0, 1.0))
    w = w[:max(1, int((w >= m32).sum()))]
    ids = order[:len(w)]
    by = np.argsort(ids)
    ids, w = ids[by], w[by]
    upto, goal = np.cumsum(w, dtype=np.longdouble), float(np.float32(u)) * w.sum(dtype=np.longdouble)
    decided &= bool(np.abs(upto - goal).min() > near) or u == 0.0
    at = min(int((upto <= goal).sum()), len(w) - 1)
    return ids[at], w[at] / w.sum(), ids, w / w.sum(), decided


def logits(rng, rows, V, kind):
    if kind == "peaked":
        x = -1.7 * np.log(1 + np.argsort(rng.random((rows, V)), 1)) + 0.3 * rng.normal(size=(rows, V))
    elif kind == "flat":
        x = 0.05 * rng.normal(size=(rows, V))
    elif kind == "normal":
        x = 3 * rng.normal(size=(rows, V))
    elif kind == "ties":
        x = rng.integers(-3, 4, size=(rows, V)) * 0.5
    elif kind == "equal":
        x = np.full((rows, V), -1.25)
    elif kind == "barred":
        x = np.where(rng.random((rows, V)) < 0.9, -np.inf, 3 * rng.normal(size=(rows, V)))
    else:
        raise AssertionError(kind)
    return x.astype(np.float32)


SETTINGS = [dict(), dict(T=0.0), dict(k=1), dict(k=3), dict(k=40), dict(k=1500), dict(p=0.9), dict(p=0.3), dict(p=0.999), dict(m=0.1), dict(m=1.0), dict(T=0.7, k=50, p=0.95),
            dict(T=1.5, k=2000, p=0.8, m=0.01), dict(T=0.01, p=0.5), dict(T=30.0, p=0.97), dict(T=30.0, k=1200, p=0.9), dict(k=10 ** 9, p=1.0, m=0.0), dict(p=1e-6), dict(T=1e-30, k=7)]


def check(ctx, x, rows, uniforms, dist=True, near=NEAR):
    """rows: a setting for each row of x."""
    T, k, p, m = (np.array([s.get(n, d) for s in rows], t) for n, d, t in (("T", 1.0, np.float32), ("k", 0, np.int32), ("p", 1.0, np.float32), ("m", 0.0, np.float32)))
    got = ctx.sample_rows(x, uniforms, T, k, p, m, want_dist=dist)
    left_out = 0
    for r in range(len(rows)):
        token, prob, ids, probs, decided = reference(x[r], T[r], int(k[r]), p[r], m[r], uniforms[r], near)
        if not decided:
            left_out += 1
            continue
        assert got[0][r] == token, (r, rows[r], uniforms[r], got[0][r], token)
        assert abs(got[1][r] - prob) <= 2.0 ** -23 * prob, (r, rows[r])
        if dist:
            full = np.zeros(x.shape[1])
            full[ids] = probs
            assert np.array_equal(got[2][r] > 0, full > 2.0 ** -46) or np.all(np.abs(got[2][r] - full) <= 2.0 ** -43)
            assert np.all(np.abs(got[2][r] - full) <= DIST * full + 2.0 ** -43)
    assert left_out <= max(2, len(rows) // 8), left_out


@pytest.mark.parametrize("kind", ["peaked", "flat", "normal", "ties", "equal", "barred"])
@pytest.mark.parametrize("V", [1, 2, 31, 777, 5003, 32000])
def test_every_filter(ctx, kind, V):
    rng = np.random.default_rng(V)
    rows = SETTINGS * 2
    check(ctx, logits(rng, len(rows), V, kind), rows, rng.random(len(rows)).astype(np.float32), near=-1 if kind == "equal" else NEAR)


@pytest.mark.parametrize("kind", ["peaked", "flat", "ties", "equal"])
def test_large_vocabulary(ctx, kind):
    rng = np.random.default_rng(3)
    rows = SETTINGS
    check(ctx, logits(rng, len(rows), 151936, kind), rows, rng.random(len(rows)).astype(np.float32), near=-1 if kind == "equal" else NEAR)


def test_the_largest_vocabulary_and_the_first_one_refused(ctx):
    rng = np.random.default_rng(4)
    rows = [dict(T=0.8, k=50, p=0.9), dict(p=0.9), dict()]
    check(ctx, logits(rng, 3, 389120, "peaked"), rows, rng.random(3).astype(np.float32), dist=False)
    with pytest.raises(dc.DcError) as e:
        ctx.sample_rows(np.zeros((1, 389121), np.float32), [0.5])
    assert e.value.status == -7


def test_draws_over_the_whole_range_of_uniforms(ctx):
    """u = 0: the first kept token with a weight; the largest u below 1: the last one; in between, shares as the probabilities."""
    rng = np.random.default_rng(5)
    x = np.tile(logits(rng, 1, 1000, "normal"), (2000, 1))
    u = ((np.arange(2000) + 0.5) / 2000).astype(np.float32)
    rows = [dict(T=0.9, k=64, p=0.95)] * 2000
    tokens, p = ctx.sample_rows(x, u, 0.9, 64, 0.95)
    _, _, ids, probs, _ = reference(x[0], 0.9, 64, 0.95, 0.0, 0.5)
    assert np.all(np.diff(tokens) >= 0)          # by index
    for i, q in zip(ids, probs):
        assert abs((tokens == i).mean() - q) <= 1.0 / 2000
    edge = np.array([0.0, np.float32(1.0) - np.float32(2.0 ** -24)], np.float32)
    assert list(ctx.sample_rows(x[:2], edge, 0.9, 64, 0.95)[0]) == [ids[0], ids[-1]]
    check(ctx, x[:40], rows[:40], u[:40])


def test_infinities_and_nan(ctx):
    rng = np.random.default_rng(6)
    V = 3001
    x = logits(rng, 8, V, "normal")
    x[0] = -np.inf                               # nothing left
    x[1] = np.nan
    x[2, ::2] = np.nan                           # NaN is never drawn
    x[3] = -np.inf
    x[3, 1234] = -3e38                           # one token
    x[4, [5, 77]] = np.inf                       # +inf: alone, evenly
    x[5] = np.finfo(np.float32).min              # a mask of the type's lowest value, everywhere
    x[6] = np.finfo(np.float32).min
    x[6, 9] = np.finfo(np.float32).max
    x[7] = 0.0
    x[7, ::2] = -0.0                             # equal values
    for s in (dict(), dict(T=0.0), dict(k=20), dict(p=0.9), dict(T=0.6, k=1300, p=0.7), dict(m=0.2)):
        u = rng.random(8).astype(np.float32)
        with np.errstate(invalid="ignore"):
            got = ctx.sample_rows(x, u, *(s.get(n, d) for n, d in (("T", 1.0), ("k", 0), ("p", 1.0), ("m", 0.0))), want_dist=True)
        assert got[0][0] == -1 and got[0][1] == -1 and not got[2][:2].any() and not got[1][:2].any()
        assert got[0][2] % 2 == 1 and got[0][3] == 1234 and got[1][3] == 1
        assert got[0][4] in (5, 77) and got[0][4] == (5 if u[4] < 0.5 or s.get("T") == 0 or s.get("p", 1) <= 0.5 else 77)
        assert got[0][6] == 9
        rest = [2, 5, 7]
        check(ctx, x[rest], [s] * 3, u[rest])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_device_rows_strides_and_missing_settings(ctx, dtype):
    rng = np.random.default_rng(7)
    rows, V, ld = 9, 4097, 4111
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    wide = torch.full((rows * ld + 1,), float("nan"), dtype=t, device=GPU)
    view = wide[1:].view(rows, ld)[:, :V]
    view.copy_(torch.from_numpy(logits(rng, rows, V, "peaked")))
    x = view.float().cpu().numpy()
    u = torch.rand(rows, device=GPU)
    tokens = torch.full((rows + 1,), -9, dtype=torch.int32, device=GPU)
    p = torch.full((rows + 1,), -9.0, device=GPU)
    dist = torch.full((rows * V + 3,), -9.0, device=GPU)
    settings = {"T": torch.full((rows,), 0.7, device=GPU), "k": torch.full((rows,), 30, dtype=torch.int32, device=GPU), "p": torch.full((rows,), 0.9, device=GPU),
                "m": torch.full((rows,), 0.02, device=GPU)}
    torch.cuda.synchronize()
    for given in ("", "T", "k", "Tk", "p", "Tp", "m", "Tkpm"):
        at = [settings[n].data_ptr() if n in given else 0 for n in "Tkpm"]
        ctx.sample_rows_dev(view.data_ptr(), rows, V, *at, u.data_ptr(), tokens.data_ptr(), p=p.data_ptr(), dist=dist.data_ptr(), ld=ld, dtype=dtype)
        ctx.synchronize()
        for r in range(rows):
            v = {n: float(settings[n][r]) for n in given}
            token, prob, ids, probs, decided = reference(x[r], v.get("T", 1.0), int(v.get("k", 0)), v.get("p", 1.0), v.get("m", 0.0), float(u[r]))
            if decided:
                assert int(tokens[r]) == token and abs(float(p[r]) - prob) <= 2.0 ** -23 * prob, (given, r)
                full = np.zeros(V)
                full[ids] = probs
                assert np.all(np.abs(dist[r * V:(r + 1) * V].cpu().numpy() - full) <= DIST * full + 2.0 ** -43)
    assert int(tokens[rows]) == -9 and float(p[rows]) == -9 and torch.all(dist[rows * V:] == -9)
    # results that are not asked for
    first = tokens.clone()
    tokens.fill_(-9)
    torch.cuda.synchronize()
    ctx.sample_rows_dev(view.data_ptr(), rows, V, *at, u.data_ptr(), tokens.data_ptr(), ld=ld, dtype=dtype)
    ctx.synchronize()
    assert torch.equal(first, tokens)


def test_many_rows_and_no_rows(ctx):
    rng = np.random.default_rng(8)
    rows = [SETTINGS[i % len(SETTINGS)] for i in range(600)]
    check(ctx, logits(rng, 600, 1009, "peaked"), rows, rng.random(600).astype(np.float32))
    ctx.sample_rows_dev(0, 0, 10, 0, 0, 0, 0, 0, 0)


def test_the_distribution_serves_a_stochastic_verification(ctx):
    """A draft's distribution after its filters as the q of the accept step: a drafted token has q > 0, so that u q < p decides."""
    rng = np.random.default_rng(9)
    V = 500
    draft = logits(rng, 3, V, "normal")
    tokens, p, q = ctx.sample_rows(draft, rng.random(3), 0.8, 20, 0.9, want_dist=True)
    assert np.all(q[np.arange(3), tokens] == p) and np.allclose(q.sum(1), 1, atol=1e-6)
    target = np.concatenate([draft, draft[:1]])
    n, nxt = ctx.verify_accept(target, tokens, q, uniforms=np.zeros(4, np.float32), mode=1, temperature=0.8)
    assert n == 3 and 0 <= nxt < V


def test_captured_and_replayed(ctx):
    rng = np.random.default_rng(10)
    x = torch.from_numpy(logits(rng, 4, 3000, "peaked")).to(GPU)
    u, tokens = torch.rand(4, device=GPU), torch.zeros(4, dtype=torch.int32, device=GPU)
    stream = torch.cuda.ExternalStream(dc._lib.lib().dc_b200_stream(ctx.handle))
    torch.cuda.synchronize()
    call = lambda: ctx.sample_rows_dev(x.data_ptr(), 4, 3000, 0, 0, 0, 0, u.data_ptr(), tokens.data_ptr())
    call()
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(5):
        x.copy_(torch.from_numpy(logits(rng, 4, 3000, "normal")))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        got = tokens.cpu().numpy().copy()
        call()
        ctx.synchronize()
        assert np.array_equal(got, tokens.cpu().numpy())
    del graph


def test_refusals(ctx):
    x = np.zeros((2, 10), np.float32)
    for bad in (dict(uniforms=1.0), dict(uniforms=-0.1), dict(uniforms=np.nan), dict(temperature=-1.0), dict(temperature=np.nan), dict(top_k=-1), dict(top_p=0.0), dict(top_p=np.nan),
                dict(min_p=1.5), dict(min_p=-0.5), dict(min_p=np.nan)):
        with pytest.raises(dc.DcError) as e:
            ctx.sample_rows(x, **({"uniforms": 0.5} | bad))
        assert e.value.status == -1
    for status, args, kw in ((-1, (256, 1, 0, 0, 0, 0, 0, 256, 256), {}), (-1, (256, -1, 5, 0, 0, 0, 0, 256, 256), {}), (-1, (0, 1, 5, 0, 0, 0, 0, 256, 256), {}),
                             (-1, (256, 1, 5, 0, 0, 0, 0, 0, 256), {}), (-1, (256, 1, 5, 0, 0, 0, 0, 256, 0), {}), (-1, (256, 1, 5, 0, 0, 0, 0, 256, 256), dict(ld=4)),
                             (-7, (256, 1, 5, 0, 0, 0, 0, 256, 256), dict(dtype="f16"))):
        with pytest.raises(dc.DcError) as e:
            ctx.sample_rows_dev(*args, **kw)
        assert e.value.status == status
    with pytest.raises(ValueError):
        ctx.sample_rows_dev(256, 1, 5, 0, 0, 0, 0, 256, 256, dtype="int8")
