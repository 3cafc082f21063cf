"""The experts' gradient of the input (csrc/moe.hip): dx[t] = sum over the
token's pairs of weight * (q(d out[t]) W_e) is summed in FP32 and rounded to the
gradients' type once, whatever that type holds."""
import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B
from test_gpu_moe import choices
from test_gpu_mx4 import ROUNDING, TYPES, normal, stored, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tokens", [3, 100, 700])
def test_dx_of_pairs_beyond_the_range_of_its_type(type, tokens):
    # a pair's product is 64 * 64 * 64 = 2^18, above FP16's range, in every
    # element; its weight brings it back, or is 0, or another pair's product of
    # the other sign cancels it.  All sums are exact.
    n = inputs = 64
    w = np.full((3, n, inputs), 64.0, np.float32)
    w[1] = -64.0
    x = np.ones((tokens, inputs), np.float32)
    dy = np.full((tokens, n), 64.0, np.float32)
    ids = np.tile(np.array([[0, 2]], np.int32), (tokens, 1))
    weights = np.tile(np.array([[2.0**-6, 0.0]], np.float32), (tokens, 1))
    ids[1::3], weights[1::3] = [0, 1], [1.0, 0.75]
    ids[2::3], weights[2::3] = [2, 1], [1.0, 1.0]
    want = np.full((tokens, 1), 2.0**12)
    want[1::3], want[2::3] = 2.0**16 if type != B.TYPE_F16 else 0.0, 0.0
    if type == B.TYPE_F16:
        weights[1::3] = [1.0, 1.0]  # 2^16 itself is beyond it
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    layer.forward(x, ids, weights)
    dx, _, _ = layer.backward(stored(dy, type)[0], type, type)
    assert np.array_equal(values(dx, type), np.broadcast_to(want, (tokens, inputs)))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tokens,k,experts,inputs,n", [(5, 8, 16, 130, 70), (16, 4, 8, 96, 200), (70, 2, 5, 130, 257),
                                                       (200, 6, 16, 300, 129)])
def test_dx_is_rounded_once(type, tokens, k, experts, inputs, n):
    # n products and k pairs summed in FP32 in any order, as in product_bound,
    # and half a unit in the last place of the output (2^-25: FP16's subnormals)
    rng = np.random.default_rng(tokens * k + n)
    raw, x = stored(normal(rng, tokens, inputs), type)
    wraw, w = stored(normal(rng, experts, n, inputs), type)
    draw, dy = stored(normal(rng, tokens, n) * 1e-2, type)
    ids, weights = choices(rng, tokens, k, experts, skew=False)
    layer = B.MoeLinear(*B.mx4_encode(wraw, type, columns=True))
    layer.forward(raw, ids, weights, type)
    got = values(layer.backward(draw, type, type)[0], type)
    want = R.experts_layer(x, ids, weights, w, dy)[2]
    real = (ids >= 0) & (ids < experts)
    wt = np.stack([np.abs(R.rounded(np.ascontiguousarray(w[e].T))) for e in range(experts)])
    z = np.einsum("tn,tjin->tji", np.abs(R.rounded(dy)), wt[np.where(real, ids, 0)]) * real[..., None]
    size = (weights[..., None] * z).sum(1)
    assert (np.abs(got - want) <= (n + k) * 2.0**-23 * size + ROUNDING[type] * np.abs(want) + 2.0**-25).all()
