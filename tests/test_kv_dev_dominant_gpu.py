"""Attention over the 16-bit cache where one key is far ahead of tens of thousands of others and has a value of 0, so that a row's answer is the others' alone."""
import pytest
import torch

from kv_dev_util import GPU, Mirror

pytestmark = pytest.mark.gpu


def run(ctx, dtype, spread, ahead, steps):
    """Scores: the first key's `ahead` (in natural units), the others' around 0, of the given spread; values around 1.  The bounds are those of the other tests, relative to the weighted
    sizes of the values: so to the others', of whom each is only e^-ahead of the first."""
    n, hd = 30000, 64
    m = Mirror(ctx, dtype, 4, 2, hd, 2, 2000, 1950, n + 200, seed=ahead)

    def keys(T):
        k = 0.5 * m.rows(T, 2).float() if spread else torch.zeros(T, 2, hd)
        k[..., 0] = 0.0
        return k.to(m.rows(1, 1).dtype)

    def values(T):
        return (1.0 + 0.5 * m.rows(T, 2).float()).to(m.rows(1, 1).dtype)

    def queries(T):
        q = m.rows(T, 4).float()
        q[..., 0] = 8.0
        return q.to(m.rows(1, 1).dtype)
    m.step([n, 3])
    T = len(m.steps.seqs)
    k, v = keys(T), values(T)
    k[0], v[0] = 0.0, 0.0
    k[0, :, 0] = ahead      # (times 8 / 8)
    kd, vd = k.to(GPU), v.to(GPU)
    torch.cuda.synchronize()
    m.cache.write_dev(0, kd.data_ptr(), vd.data_ptr())
    ctx.synchronize()
    m.append(0, k, v)
    for count, window, keep in steps:
        m.step(count)
        T = len(m.steps.seqs)
        m.attend(q=queries(T), k=keys(T), v=values(T), window=window, keep=keep)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spread", [0.5, 0.0])
@pytest.mark.parametrize("ahead", [12, 14, 16, 18, 22])
def test_the_rest_beside_a_dominant_key(ctx, dtype, spread, ahead):
    """Single tokens and drafted ones; f32 prompts."""
    run(ctx, dtype, spread, ahead, (([1, 1], 0, 0), ([5, 0], 0, 0), ([1, 0], 20000, 1), ([34 if dtype == "f32" else 16, 0], 0, 0)))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("spread", [0.5, 0.0])
@pytest.mark.parametrize("ahead", [12, 14, 16, 18, 22])
def test_the_rest_beside_a_dominant_key_of_prompts(ctx, dtype, spread, ahead):
    run(ctx, dtype, spread, ahead, (([34, 0], 0, 0), ([70, 1], 20000, 1)))
