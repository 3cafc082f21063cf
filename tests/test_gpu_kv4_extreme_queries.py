"""Queries at the ends of their type's range, in both kernels of the attention over
the paged MX4 cache."""
import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_kv4 import attend, check_attention, tables

pytestmark = pytest.mark.gpu

LARGEST = {B.TYPE_F32: float(np.finfo(np.float32).max), B.TYPE_BF16: float(2**127 * (2 - 2.0**-7)), B.TYPE_F16: 65504.0}
TYPES = [(B.TYPE_F32, B.TYPE_F32), (B.TYPE_BF16, B.TYPE_F32), (B.TYPE_F32, B.TYPE_BF16), (B.TYPE_F16, B.TYPE_F16),
         (B.TYPE_BF16, B.TYPE_BF16)]


def small_keys(rng, pages, dim, positive=()):
    """A cache of keys of some 2^-12, those of the channels `positive` above zero."""
    c = K.Cache(pages, 16, 1, dim)
    for s in range(pages * 16):
        k = rng.uniform(0.25, 1.0, (1, dim))
        k *= np.where(np.isin(np.arange(dim), positive), 1.0, rng.choice([-1.0, 1.0], dim))
        c.put(s, k * 2.0**-12, rng.standard_normal((1, dim)))
    return c


@pytest.mark.parametrize("type,out_type", TYPES)
@pytest.mark.parametrize("count,group,dim", [(1, 2, 64), (5, 3, 128), (80, 1, 64), (40, 2, 33)])
def test_the_largest_finite_queries(type, out_type, count, group, dim):
    # values from a quarter of the type's largest to the largest itself, and the
    # FP32 ones around the middle between BF16's largest and infinity
    rng = np.random.default_rng(dim + count)
    c, most = small_keys(rng, 8, dim), LARGEST[type]
    q = rng.uniform(0.25, 1.0, (count, group, dim)) * most
    q[:, :, ::3] = most
    if type == B.TYPE_F32:
        middle = 2.0**127 * (2 - 2.0**-8)
        q[:, :, 1], q[:, :, 4], q[:, :, 7] = middle, middle - 2.0**104, middle + 2.0**104
    q *= rng.choice([-1.0, 1.0], q.shape)
    lengths, counts = [100], [count]
    check_attention(c, tables(rng, c, lengths, 7), lengths, counts, q, 2.0**11 / most, type, out_type)


@pytest.mark.parametrize("exponent", [100, 112, 119, 122])
@pytest.mark.parametrize("count", [1, 80])
def test_the_smallest_queries(count, exponent):
    # against keys as large: an FP32 query's last piece is a multiple of BF16's
    # smallest step, so it is off by up to half of 2^-133, times a key in each channel
    rng = np.random.default_rng(exponent)
    c = K.Cache(8, 16, 1, 32)
    for s in range(128):
        c.put(s, rng.choice([-1.0, 1.0], (1, 32)) * rng.uniform(0.25, 1.0, (1, 32)) * 2.0**exponent, rng.standard_normal((1, 32)))
    q = (rng.uniform(0.5, 1.0, (count, 1, 32)) * rng.choice([-1.0, 1.0], (count, 1, 32)) * 2.0**-exponent).astype(np.float32)
    got, lse = attend(c, np.arange(8)[None], [128], [count], q, 1.0, 0, 0)
    want, want_lse, of = K.attention(c, np.arange(8), 128, q.astype(np.float64), 1.0)
    bound, lse_bound, _ = K.attention_bound(of, 128, 32, 3, 0)
    off = 2.0**-134 * np.abs(c.values(0)).sum(2).max()
    assert (np.abs(got - want) <= bound + 2 * off * of[0] + 2.0**-24 * np.abs(want)).all()
    assert (np.abs(lse - want_lse) <= lse_bound + off).all()


@pytest.mark.parametrize("type,out_type", TYPES)
@pytest.mark.parametrize("count", [6, 90])
def test_infinite_queries(type, out_type, count):
    # infinity times a key is infinite or NaN, so the softmax over any keys is NaN,
    # also where all scores are minus infinity; a query that sees no key stays zero
    rng = np.random.default_rng(count)
    c = small_keys(rng, 8, 64, positive=(3, 40))
    q = rng.standard_normal((count, 2, 64)) * 100
    q[0, 0, 3], q[count - 1, 1, 3] = -np.inf, -np.inf
    q[count - 2, 0, 40], q[count - 3, 1, 40] = np.inf, np.nan
    q[count - 4, 0, 5], q[count - 4, 1, 5] = -np.inf, np.inf
    for length in (100, 3):  # of three keys the first queries see none
        for scale in (0.1, -0.1):
            got, lse, _ = check_attention(c, tables(rng, c, [length], 7), [length], [count], q, scale, type, out_type)
            bad = np.isnan(lse)
            assert bad.sum() == (6 if length == 100 else 3)
            assert (np.isnan(got).all(2) == bad).all()
    assert (got[: count - 3] == 0).all()
