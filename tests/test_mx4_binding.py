"""The Python binding of the MX4 and expert-layer calls refuses arrays and packed
matrices whose sizes do not agree, before anything is uploaded: the C calls see
only pointers.  Without a GPU."""
import numpy as np
import pytest

import bitsqz_amd as B


class Untouched:
    """In the place of device memory: nothing may be asked of it."""

    def __init__(self, nbytes):
        raise AssertionError("device memory was asked for")

    @staticmethod
    def from_array(a):
        raise AssertionError("an upload was asked for")


def packed(rows, cols, batch=1):
    m = object.__new__(B.Mx4)
    m.rows, m.cols, m.batch, m.codes, m.scales = rows, cols, batch, None, None
    return m


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    monkeypatch.setattr(B, "DeviceBuffer", Untouched)


def refused(call, word):
    with pytest.raises(ValueError, match=word):
        call()


def zeros(*shape):
    return np.zeros(shape, np.float32)


def ids(*shape):
    return np.zeros(shape, np.int32)


def test_encode():
    refused(lambda: B.mx4_encode(zeros(8)), "rows x cols")
    refused(lambda: B.mx4_encode(zeros(2, 2, 2, 8)), "rows x cols")


def test_product():
    refused(lambda: B.mx4_product(packed(4, 64), packed(5, 65)), "columns")
    refused(lambda: B.mx4_product(packed(4, 64), packed(5, 64, batch=3)), "batch")
    refused(lambda: B.mx4_product(packed(4, 64, batch=2), packed(5, 64)), "batch")


def test_linear():
    refused(lambda: B.mx4_linear(zeros(4, 63), packed(5, 64)), "columns")
    refused(lambda: B.mx4_linear(zeros(4, 64), packed(5, 64, batch=2)), "batch")
    refused(lambda: B.mx4_linear(zeros(64), packed(5, 64)), "matrix")


@pytest.mark.parametrize("dy,xt,wt,word", [
    ((4, 5), (64, 3), (64, 5), "kept columns"), ((4, 5), (64, 4), (64, 6), "weights' columns"),
    ((4, 5), (65, 4), (64, 5), "inputs"), ((4, 5), (64, 4, 2), (64, 5), "batch"), ((4, 5), (64, 4), (64, 5, 2), "batch"),
    ((5,), (64, 4), (64, 5), "matrix"),
])
def test_linear_backward(dy, xt, wt, word):
    refused(lambda: B.mx4_linear_backward(zeros(*dy), packed(*xt), packed(*wt)), word)


def test_route():
    refused(lambda: B.moe_route(zeros(4, 8), 2, bias=zeros(7)), "bias")
    refused(lambda: B.moe_route(zeros(4, 8), 2, bias=zeros(4, 8)), "bias")
    refused(lambda: B.moe_route(zeros(8), 2), "matrix")
    refused(lambda: B.moe_route_backward(zeros(4, 8), ids(3, 2), zeros(3, 2)), "ids")
    refused(lambda: B.moe_route_backward(zeros(4, 8), ids(4, 2), zeros(4, 3)), "weights")
    refused(lambda: B.moe_route_backward(zeros(4, 8), ids(4, 2), zeros(3, 2)), "weights")
    refused(lambda: B.moe_route_backward(zeros(4, 8), ids(4), zeros(4)), "ids")


def test_layer():
    w, wt = packed(8, 64, batch=3), packed(64, 8, batch=3)
    for other in (packed(64, 8, batch=2), packed(63, 8, batch=3), packed(64, 9, batch=3)):
        refused(lambda: B.MoeLinear(w, other), "weights' columns")
    layer = B.MoeLinear(w, wt)
    refused(lambda: layer.forward(zeros(4, 63), ids(4, 2), zeros(4, 2)), "columns")
    refused(lambda: layer.forward(zeros(64), ids(4, 2), zeros(4, 2)), "matrix")
    refused(lambda: layer.forward(zeros(4, 64), ids(3, 2), zeros(3, 2)), "ids")
    refused(lambda: layer.forward(zeros(4, 64), ids(4), zeros(4)), "ids")
    refused(lambda: layer.forward(zeros(4, 64), ids(4, 2), zeros(4, 1)), "weights")
    refused(lambda: layer.backward(zeros(4, 8)), "forward")


def test_layer_backward():
    w = packed(8, 64, batch=3)
    layer = B.MoeLinear(w)
    layer.m, layer.k, layer.done = 4, 2, True  # as a forward call leaves them
    refused(lambda: layer.backward(zeros(4, 8)), "weights' columns")
    layer.wt = packed(64, 8, batch=3)
    refused(lambda: layer.backward(zeros(4, 9)), "d_out")
    refused(lambda: layer.backward(zeros(5, 8)), "d_out")
    refused(lambda: layer.backward(zeros(32)), "matrix")


def test_a_refused_forward_leaves_nothing_to_go_back_through():
    layer = B.MoeLinear(packed(8, 64, batch=3), packed(64, 8, batch=3))
    layer.m, layer.k, layer.done = 4, 2, True
    refused(lambda: layer.forward(zeros(4, 63), ids(4, 2), zeros(4, 2)), "columns")
    refused(lambda: layer.backward(zeros(4, 8)), "forward")
