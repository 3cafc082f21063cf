"""Attention over the paged MX4 cache with tables of the largest size that a call
takes: 2^31 - 48 keys in pages of 16, most of them one page, and a window, so that
only the last keys count."""
import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_kv4 import attend, filled, stored

pytestmark = pytest.mark.gpu

WIDTH = (2**31 - 1 - 32) // 16


@pytest.mark.parametrize("short", [0, 15, 16])  # of the table's end; the last block of 64 keys ends past 31 bits but for the last
@pytest.mark.parametrize("count", [1, 40])      # a single token, a prompt
def test_the_last_keys_of_the_longest_table(count, short):
    rng = np.random.default_rng(count + short)
    c = filled(rng, 14, 16, 1, 64)
    tail = rng.permutation(13)[:12] + 1
    table = np.zeros((1, WIDTH), np.int32)
    table[0, -12:] = tail
    q = rng.standard_normal((count, 2, 64))
    raw, q64 = stored(q, B.TYPE_F32)
    got, lse = attend(c, table, [WIDTH * 16 - short], [count], raw, 0.1, 0, 0, window=100)
    # the last 12 pages hold all that any query sees
    want, want_lse, of = K.attention(c, tail, 192 - short, q64, float(np.float32(0.1)), window=100)
    bound, lse_bound, _ = K.attention_bound(of, 192, 64, 3, 0)
    assert (np.abs(got - want) <= bound + 2.0**-24 * np.abs(want)).all()
    assert (np.abs(lse - want_lse) <= lse_bound).all()
