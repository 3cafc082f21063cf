"""Attention over the paged MX4 cache at scales near zero, with scores near FP32's
largest."""
import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_kv4 import check_attention, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", [B.TYPE_F32, B.TYPE_BF16])
@pytest.mark.parametrize("count", [1, 80])
@pytest.mark.parametrize("scale", [0.0, 1e-44, -1e-40, 2e-38])
def test_scales_near_zero(scale, count, type):
    # scores of up to some 2^125 before their scale; a scale of zero weighs all keys alike
    rng = np.random.default_rng(count)
    c = K.Cache(8, 16, 1, 64)
    for s in range(128):
        c.put(s, rng.uniform(0.25, 1.0, (1, 64)) * rng.choice([-1.0, 1.0], (1, 64)), rng.standard_normal((1, 64)))
    q = rng.uniform(0.25, 1.0, (count, 2, 64)) * rng.choice([-1.0, 1.0], (count, 2, 64)) * 2.0**122
    check_attention(c, tables(rng, c, [100], 7), [100], [count], q, scale, type)
