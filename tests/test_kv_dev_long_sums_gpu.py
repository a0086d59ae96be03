"""f32 results of attention over many pages a warp: rounding errors of the sums do not add up in one direction."""
import pytest
import torch

from kv_dev_util import GPU, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv,new,window,keep", [(2, 1, 40, 0, 0), (4, 1, 70, 20000, 100), (128, 128, 1, 0, 0), (64, 32, 3, 0, 0)])
def test_answers_of_long_sequences(ctx, hd, heads, kv, new, window, keep):
    """30000 positions, values around 1, scores within a few units.  A row's relative error: queries, weights and exponentials 2^-22 each, scores of some units 2^-22 of them, and sums of n pages that are
    rounded to nearest: sqrt(n) 2^-25, of both the answers and the weights.  Together below 2^-19 of the norm; n errors of one direction, 2^-25 each, would be some 2^-14 for the prompts."""
    before, g = 30000, torch.Generator(GPU).manual_seed(heads + hd)
    pages = -(-(before + new) // 16)
    cache = ctx.kv_cache_dev(1, heads, kv, hd, pages, 1, pages, before, dtype="f32")
    normal = lambda *s: torch.randn(*s, generator=g, device=GPU)  # noqa: E731
    k, v = (0.5 * normal(before + new, kv, hd)), 1.0 + 0.3 * normal(before + new, kv, hd)
    q, out = normal(new, heads, hd), torch.empty(new, heads, hd, device=GPU)
    counts = [ints([before]), ints([new])]
    torch.cuda.synchronize()
    cache.step_dev(counts[0].data_ptr(), max_count=before)
    cache.write_dev(0, k.data_ptr(), v.data_ptr())
    cache.step_dev(counts[1].data_ptr(), max_count=new)
    cache.attend_dev(0, q.data_ptr(), k[before:].data_ptr(), v[before:].data_ptr(), hd ** -0.5, out.data_ptr(), window=window, keep_first=keep)
    ctx.synchronize()
    G = heads // kv
    at, row = torch.arange(before + new, device=GPU)[None], torch.arange(before, before + new, device=GPU)[:, None]
    sees = (at <= row) & ((at > row - window) | (at < keep)) if window else at <= row
    off, size = 0.0, 0.0
    for h in range(heads):
        z = (q[:, h].double() @ k[:, h // G].half().double().T * hd ** -0.5).masked_fill(~sees, -float("inf"))
        y = torch.softmax(z, -1) @ v[:, h // G].half().double()
        off, size = off + float((out[:, h].double() - y).square().sum()), size + float(y.square().sum())
    cache.close()
    assert (off / size) ** 0.5 <= 2.0**-19, (off / size) ** 0.5
