"""Verified tokens of shallow rows over a large vocabulary, where most tokens have a share of a millionth and less: every accepted draft and every drawn token is the one that 64 bits give.

Weights of a sum are within 2^-46 of themselves on either side, and errors of some 10^5 of them have both signs: a border between two tokens is off by some 2^-50 of the whole, where some
10^5 draws, with 1.5 10^5 borders each, meet one in fewer than one of 10^4 runs."""
import numpy as np
import pytest
import torch

from kv_dev_util import GPU

pytestmark = pytest.mark.gpu
V = 151936
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def rows_of(n, dtype, seed, steep=1.0):
    """Logits that fall with a power of the rank."""
    g = torch.Generator(GPU).manual_seed(seed)
    ranked = 9.0 - steep * torch.log(torch.arange(1, V + 1, device=GPU).float())
    x = torch.stack([ranked[torch.randperm(V, generator=g, device=GPU)] for _ in range(n)])
    return (x + 0.3 * torch.randn(n, V, generator=g, device=GPU)).to(TYPES[dtype])


def shares(x, T):
    x = x.double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / float(np.float32(T)))      # (the call takes f32 temperatures)
    return w / w.sum(-1, keepdim=True)


def drawn(w, u):
    """First token, by index, up to which the sum is above u times the whole; a row of w a number."""
    upto = w.cumsum(-1)
    return torch.searchsorted(upto, (u.double()[:, None] * upto[:, -1:]).contiguous(), right=True)[:, 0]


def call(ctx, x, starts, tokens, q, u, T, probs=False):
    D, R = tokens.shape
    out = torch.full((R, D + 1), -9, dtype=torch.int32, device=GPU)
    acc, rej = torch.full((R,), -9, dtype=torch.int32, device=GPU), torch.full((R,), -9, dtype=torch.int32, device=GPU)
    T = torch.full((R,), T, device=GPU)
    torch.cuda.synchronize()
    ctx.verify_rows_dev(x.data_ptr(), R, V, D, tokens.data_ptr() if D else 0, q.data_ptr() if q is not None else 0, u.data_ptr(), out.data_ptr(), acc.data_ptr(), rejected=rej.data_ptr(),
                        starts=starts.data_ptr(), temperature=0 if probs else T.data_ptr(), rows=len(x), dtype="bf16" if x.dtype == torch.bfloat16 else "f32", probs=probs)
    ctx.synchronize()
    assert torch.equal(rej, D - acc)
    return out, acc


def i32(x):
    return x.to(torch.int32).contiguous()


@pytest.mark.parametrize("dtype,T", [("bf16", 1.0), ("bf16", 1.3), ("f32", 0.7), ("f32", 1.3), ("probs", 1.0)])
def test_tokens_drawn_from_the_target(ctx, dtype, T):
    n, R = 16, 8192
    x = rows_of(n, "f32" if dtype == "probs" else dtype, 1)
    if dtype == "probs":
        x = torch.softmax(x, -1)
    g = torch.Generator(GPU).manual_seed(2)
    u = torch.rand(R, 1, generator=g, device=GPU)
    starts = i32(torch.arange(R, device=GPU) % n)
    out, acc = call(ctx, x, starts, torch.zeros(0, R, dtype=torch.int32, device=GPU), None, u, T, probs=dtype == "probs")
    p = x.double() if dtype == "probs" else shares(x, T)
    for s in range(n):
        of = torch.arange(s, R, n, device=GPU)
        assert torch.equal(out[of, 0].long(), drawn(p[s].expand(len(of), V), u[of, 0])), s


@pytest.mark.parametrize("dtype,T", [("bf16", 1.0), ("bf16", 1.3), ("f32", 0.7), ("f32", 1.3), ("probs", 1.0)])
def test_tokens_drawn_from_what_the_draft_leaves(ctx, dtype, T):
    """A draft outside the vocabulary is not accepted, whatever its number: all draws are from max(0, p - q)."""
    R = 128
    x = rows_of(R + 1, "f32" if dtype == "probs" else dtype, 3)      # (a request has a row more than drafts)
    g = torch.Generator(GPU).manual_seed(4)
    p = shares(x, T)
    q = torch.softmax(x[:R].float() / T + 0.6 * torch.randn(R, V, generator=g, device=GPU), -1)[None].contiguous()
    if dtype == "probs":
        x = p.float()
        p = x.double()
    left = (p[:R] - q[0].double()).clamp(min=0)
    starts, tokens = i32(torch.arange(R, device=GPU)), torch.full((1, R), -1, dtype=torch.int32, device=GPU)
    for _ in range(40):
        u = torch.rand(R, 2, generator=g, device=GPU)
        out, acc = call(ctx, x, starts, tokens, q, u, T, probs=dtype == "probs")
        assert (acc == 0).all() and torch.equal(out[:, 0].long(), drawn(left, u[:, 1]))


@pytest.mark.parametrize("dtype,T", [("bf16", 1.3), ("f32", 1.0), ("probs", 1.0)])
def test_tokens_drawn_beside_a_certain_draft(ctx, dtype, T):
    n, R = 16, 4096
    x = rows_of(n + 1, "f32" if dtype == "probs" else dtype, 5)
    p = shares(x, T)
    if dtype == "probs":
        x = p.float()
        p = x.double()
    g = torch.Generator(GPU).manual_seed(6)
    starts = i32(torch.arange(R, device=GPU) % n)
    own = i32(p.argmax(-1)[starts.long()])[None]
    u = torch.rand(R, 2, generator=g, device=GPU)
    u[:, 0] = 0.999
    out, acc = call(ctx, x, starts, own, None, u, T, probs=dtype == "probs")
    assert p.max() < 0.999 and (acc == 0).all()
    for s in range(n):
        of = torch.arange(s, R, n, device=GPU)
        left = p[s].clone()
        left[own[0, s]] = 0
        assert torch.equal(out[of, 0].long(), drawn(left.expand(len(of), V), u[of, 1])), s


@pytest.mark.parametrize("dtype,T", [("bf16", 1.0), ("f32", 1.3), ("f32", 0.7), ("f32", 1e-3), ("f32", 2e-33), ("probs", 1.0)])
def test_drafts_next_to_their_border(ctx, dtype, T):
    """Uniform numbers at p / q and some of f32's neighbours of it: a draft is accepted exactly where u q < p."""
    n, R = 4, 512
    x = rows_of(n + 1, "f32" if dtype == "probs" else dtype, 7)
    p = shares(x, T)
    if dtype == "probs":
        x = p.float()
        p = x.double()
    g = torch.Generator(GPU).manual_seed(8)
    starts = torch.arange(R, device=GPU) % n
    # (tokens of some weight: a number below f32's range could not stand next to the border)
    tokens = torch.stack([torch.multinomial(p[s].float(), 1, generator=g)[0] for s in starts.tolist()])
    q = torch.zeros(1, R, V, device=GPU)
    at = torch.arange(R, device=GPU)
    q[0, at, tokens] = ((1.0 + torch.rand(R, generator=g, device=GPU)).double() * p[starts, tokens]).float()
    border = (p[starts, tokens] / q[0, at, tokens].double()).float()
    u = torch.rand(R, 2, generator=g, device=GPU)
    u[:, 0] = (border.view(torch.int32) + torch.randint(-2, 3, (R,), generator=g, device=GPU).int()).view(torch.float32).clamp(max=0.99999994)
    out, acc = call(ctx, x, i32(starts), i32(tokens)[None], q, u, T, probs=dtype == "probs")
    want = u[:, 0].double() * q[0, at, tokens].double() < p[starts, tokens]
    assert 0.1 * R < want.sum() < 0.9 * R and torch.equal(acc.bool(), want)


def test_a_draft_all_but_the_target(ctx):
    """q is p rounded to f32: what is left is the rounding alone, and the token is drawn from that (each border within 2^-20 of what is left: on either side a share p is off by some 2^-50
    of itself, and what is left of all is some 2^-26)."""
    R = 24
    x = rows_of(R + 1, "f32", 9)
    p = shares(x, 1.0)[:R]
    q = p.float()[None].contiguous()
    left = (p - q[0].double()).clamp(min=0)
    upto = left.cumsum(-1)
    g = torch.Generator(GPU).manual_seed(10)
    u = torch.rand(R, 2, generator=g, device=GPU)
    out, acc = call(ctx, x, i32(torch.arange(R, device=GPU)), torch.full((1, R), -1, dtype=torch.int32, device=GPU), q, u, 1.0)
    t, goal, off = out[:, :1].long(), u[:, 1:].double() * upto[:, -1:], 2.0**-20 * upto[:, -1:]
    before = torch.where(t > 0, upto.gather(1, (t - 1).clamp(min=0)), 0.0)
    assert (acc == 0).all() and (t >= 0).all() and (before <= goal + off).all() and (upto.gather(1, t) > goal - off).all() and (left.gather(1, t) > 0).all()
