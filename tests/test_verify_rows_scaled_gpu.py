"""Verification where logits over temperature are in the hundred thousands: what counts are differences of logits, however large they are themselves."""
import numpy as np
import pytest
import torch

from kv_dev_util import GPU

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at,T", [(300.0, 1e-3), (-70.0, 3e-4), (9.0, 1e-3), (600.0, 2e-3)])
@pytest.mark.parametrize("V", [9, 257, 5000])
def test_drafts_near_their_border(ctx, at, T, V):
    """Drafts whose u q lies 2^-13 of p on either side of it.  Sums are off by less than 2^-18, a weight is by 2^-22 and by 2^-23 for every power of two below the largest (which are below 2^6 here)."""
    g = torch.Generator("cpu").manual_seed(V)
    n, R = 40, 40 * 8
    x = (at + 5 * T * torch.randn(n + 1, V, generator=g)).float()
    d = (x.double() - x.double().amax(1, keepdim=True)) / float(np.float32(T))
    p = torch.softmax(d, 1)
    assert d.abs().max() / np.log(2) < 64
    starts, side = torch.arange(R) % n, torch.arange(R) // n % 2
    tokens = torch.stack([torch.multinomial(p[s], 1, generator=g)[0] for s in starts.tolist()])
    p = p[starts, tokens]
    u = torch.rand(R, 2, generator=g)
    q = torch.zeros(1, R, V)
    q[0, torch.arange(R), tokens] = 1.25 * p.float()
    u[:, 0] = (p * (1 + (2 * side - 1) * 2.0**-13) / q[0, torch.arange(R), tokens].double()).float()
    x, starts_d, tokens_d, q, u, Td = x.to(GPU), starts.int().to(GPU), tokens.int()[None].contiguous().to(GPU), q.to(GPU), u.to(GPU), torch.full((R,), T, device=GPU)
    out, acc = torch.full((R, 2), -9, dtype=torch.int32, device=GPU), torch.full((R,), -9, dtype=torch.int32, device=GPU)
    torch.cuda.synchronize()
    ctx.verify_rows_dev(x.data_ptr(), R, V, 1, tokens_d.data_ptr(), q.data_ptr(), u.data_ptr(), out.data_ptr(), acc.data_ptr(), starts=starts_d.data_ptr(), temperature=Td.data_ptr(), rows=n + 1)
    ctx.synchronize()
    assert acc.cpu().tolist() == (1 - side).tolist()
