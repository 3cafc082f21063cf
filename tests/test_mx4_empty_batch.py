"""A dense layer's gradients of an empty batch, through the Python binding: as
the forward call, it succeeds; nothing is summed.  Without a GPU."""
import numpy as np
import pytest

import bitsqz_amd as B
from test_mx4_binding import packed, zeros


@pytest.mark.parametrize("g", [B.TYPE_F32, B.TYPE_BF16, B.TYPE_F16])
@pytest.mark.parametrize("m,n", [(0, 5), (4, 0), (0, 0)])
def test_gradients_of_nothing_are_zeros(m, n, g):
    dx, dw = B.mx4_linear_backward(zeros(m, n), packed(64, m), packed(64, n), g_type=g)
    assert dx.shape == (m, 64) and dw.shape == (n, 64)
    assert dx.dtype == dw.dtype == {B.TYPE_F32: np.float32, B.TYPE_BF16: np.uint16, B.TYPE_F16: np.float16}[g]
    assert (dx == 0).all() and (dw == 0).all()


def test_sizes_still_have_to_agree():
    with pytest.raises(ValueError, match="kept columns"):
        B.mx4_linear_backward(zeros(0, 5), packed(64, 3), packed(64, 5))
