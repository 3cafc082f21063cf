"""The routing gradient (csrc/moe.hip) where the sum of a token's chosen scores
is at or below the smallest normal FP32 number, which is then what the weights
are over: the derivative of those weights, from differences in 64 bits.  Scores
there are subnormal, good to 2^-21 of themselves; 2^-16 of the largest gradient
is allowed, as in test_gpu_moe.py."""
import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B

pytestmark = pytest.mark.gpu


def differences(x, ids, dw, sigmoid, scale, h=1e-5):
    got = np.zeros_like(x)
    for e in range(x.shape[1]):
        up, down = x.copy(), x.copy()
        up[:, e] += h
        down[:, e] -= h
        got[:, e] = ((R.weights_of(up, ids, sigmoid, True, scale) - R.weights_of(down, ids, sigmoid, True, scale)) * dw).sum(1) / (2 * h)
    return got


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("scale", [1.0, 2.5])
@pytest.mark.parametrize("size", [1.0, 50.0])
def test_gradient_of_small_sums(sigmoid, scale, size):
    # the chosen are near -88 (exp(-87.34) is the smallest normal); for softmax
    # an expert that is not among them has nearly the whole sum, as where a bias
    # chooses
    low = np.array([[-88.25, -88.5, -88.625], [-88.0, -100.0, -101.0], [-87.0, -88.0, -86.5], [-86.0, -80.0, -88.5],
                    [-88.5, -88.5, -88.5], [-3.0, -2.0, -88.0]])
    x = np.concatenate([low, np.full((len(low), 3), -200.0 if sigmoid else 0.0)], 1)
    if not sigmoid:
        x[:, 4:] = -200.0
    x = np.ascontiguousarray(x.astype(np.float32).astype(np.float64))
    ids = np.tile(np.array([[1, 0, 2]], np.int32), (len(x), 1))
    ids[1] = [0, -1, -1]
    dw = (np.array([[1.0, -0.5, 0.25]]) * size).astype(np.float32).repeat(len(x), 0)
    want = differences(x, ids, dw, sigmoid, scale)
    got = B.moe_route_backward(x, ids, dw, B.TYPE_F32, int(sigmoid), True, scale)
    assert (np.abs(got - want) <= 2.0**-16 * size * scale).all(), (got, want)
