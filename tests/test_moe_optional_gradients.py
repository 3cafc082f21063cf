"""The experts' backward call with some of its gradients left out
(include/bitsqz_llm_c.h, group 6): what only those need is not looked at."""
import numpy as np
import pytest

import bitsqz_amd as B
from test_mx4_refusals import D, refused


def back(size, m=4, n=8, ldd=8, x=D, inputs=300, ldx=300, wt=D, y=D, dx=D, lddx=300, dweights=D, dw=D):
    return B.lib().bsq_moe_linear_backward(D, 0, m, n, ldd, x, 0, inputs, ldx, D, D, 2, D, D, y, 0, wt, wt, 5, dx, lddx,
                                           dweights, dw, 0, D, size, None)


def test_row_distances_of_what_is_not_asked_for():
    # each call is refused for its workspace, the last thing that is checked
    need = B.lib().bsq_moe_linear_backward_workspace(4, 2, 8, 300, 5)
    refused(back(need - 1, dx=None, wt=None, lddx=0), "workspace")
    refused(back(need - 1, dw=None, x=None, ldx=0), "workspace")
    refused(back(need - 1, dweights=None, y=None), "workspace")
    refused(back(need, lddx=299), "overlap")
    refused(back(need, ldx=299), "overlap")
    refused(back(need, dx=None, dw=None, ldd=7), "overlap")


@pytest.mark.gpu
def test_gradients_by_themselves():
    rng = np.random.default_rng(12)
    tokens, k, experts, inputs, n = 40, 2, 5, 140, 75
    x, w, dy = (rng.standard_normal(s).astype(np.float32) for s in ((tokens, inputs), (experts, n, inputs), (tokens, n)))
    ids = np.stack([rng.choice(experts, k, replace=False) for _ in range(tokens)]).astype(np.int32)
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    layer.forward(x, ids, rng.random((tokens, k)).astype(np.float32))
    whole = layer.backward(dy)
    L, d = B.lib(), B.DeviceBuffer.from_array(dy)
    work = B.DeviceBuffer(L.bsq_moe_linear_backward_workspace(tokens, k, n, inputs, experts))
    outs = [B.DeviceBuffer(v.nbytes) for v in whole]
    for only in range(3):
        dx, dweights, dw = (outs[i].ptr if i == only else None for i in range(3))
        B.check(L.bsq_moe_linear_backward(
            d.ptr, 0, tokens, n, n, layer.x.ptr if dw else None, 0, inputs, inputs if dw else 0, layer.ids.ptr,
            layer.weights.ptr, k, layer.offsets.ptr, layer.order.ptr, layer.y.ptr if dweights else None, 0,
            layer.wt.codes.ptr if dx else None, layer.wt.scales.ptr if dx else None, experts, dx, inputs if dx else 0,
            dweights, dw, 0, work.ptr, work.nbytes, None), "backward")
        B.check(L.bsq_stream_synchronize(None), "sync")
        assert np.array_equal(outs[only].download(np.float32, whole[only].size).reshape(whole[only].shape), whole[only])
