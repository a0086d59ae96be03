"""Attention over the cache in 4 bits where one key has nearly all the weight and a value near zero, so that the rest's weights decide the answer.

bf16 rows.  Few rows: weights times scales are fp16 relative to their largest, off by 2^-11 of themselves or by 2^-25 of it, times codes up to 15.  Portions of 64 rows or
more: weights are fp16 with the largest at 2^7 or above, off by 2^-11 of themselves or by 2^-32 of the largest weight, values by 2^-11.  Scores here are exact up to
their rounding in f32 (2^-24 of 30) and the exponential's (2^-21): 2^-18 of a weight in all.  The result is rounded to bf16, by eps / 2."""
import numpy as np
import pytest
import torch

from test_kv_q4_gpu import Mirror, bf16, bits, held, unbits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [1, 7, 8, 40, 2500])      # of eight query heads a key head: 64 rows from eight tokens on, keys in one part from 2400 on
@pytest.mark.parametrize("below", [12.6, 20.3, 25.2, 26.4, 28.7])
def test_a_dominant_key_with_a_value_near_zero(ctx, below, count):
    rng = np.random.default_rng(int(below * 10) + count)
    hd, n = 128, 6000
    m = Mirror(ctx, "bf16", 8, 1, hd, 1, 560)
    a = m.cache.seq_alloc()
    k = np.zeros((n + count, 1, hd), np.float32)
    k[0] = 1.0
    v = bf16(np.abs(rng.normal(size=(n + count, 1, hd))))
    v[0] = bf16(v[0] * 2.0 ** -10)
    q = np.ones((count, 8, hd), np.float32)
    scale = float(np.float32(below * np.log(2.0) / hd))
    m.cache.batch([a], [0], [n])
    m.cache.attend(0, bits(np.zeros((n, 8, hd), np.float32)), bits(k[:n]), bits(v[:n]), scale)
    m.cache.batch([a], [n], [count])
    out = unbits(m.cache.attend(0, bits(q), bits(k[n:]), bits(v[n:]), scale))
    V = held(v)
    first = np.exp(scale * hd)                                                          # weight of the first key, the others' are 1
    total = np.cumsum(np.concatenate([first * V[:1].astype(np.float64), V[1:]]), axis=0)[n:]
    y = np.repeat(total / (first + np.arange(n, n + count))[:, None, None], 8, axis=1)
    s, most = V.reshape(n + count, 2, 64), np.abs(V).max()
    steps = (s.max(-1) - s.min(-1)).max(-1) / 15                                       # (of codes, at least the scale less its rounding)
    w = np.exp2(np.where(np.arange(n + count) == 0, 0.0, -below))
    if count * 8 >= 64:
        tol = (n + count) * 2.0 ** -32 * most + (2.0 ** -10 + 2.0 ** -18) * y
    else:
        tol = (n + count) * 15 * 2.0 ** -25 * (w * steps).max() * 1.01 + (2.0 ** -11 + 2.0 ** -18) * y
    tol = tol + (y + tol) * torch.finfo(torch.bfloat16).eps / 2
    assert np.abs(out / y - 1).max() < 1 and np.all(np.abs(out - y) <= tol), (np.abs(out - y) / tol).max()
