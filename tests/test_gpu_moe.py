"""Routing to experts and the experts' layer (csrc/moe.hip, csrc/mx4_gemm.hip)
against their definitions in 64 bits (_mx4ref.py).

Ids are compared wherever the keys that decide a token's choice lie further
apart than FP32 scores can be off (2^-20 of at most 1 plus the bias); equal
keys go to the lowest number and are compared too.  Weights: exp and a sum in
FP32, 2^-18 of a weight.  Gradients: 2^-16 of the largest magnitude that enters
a row, plus the output type's rounding.  Layers: the worst case of their FP32
sums, as in test_gpu_mx4.py."""
import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B
from test_gpu_mx4 import ROUNDING, TYPES, normal, stored, values

pytestmark = pytest.mark.gpu

LOWEST = {B.TYPE_F32: -float(np.finfo(np.float32).max), B.TYPE_BF16: -float(B.from_bf16(np.array([0x7F7F], np.uint16))[0]),
          B.TYPE_F16: -65504.0}


def check_route(raw, x, type, k, bias=None, sigmoid=False, groups=1, kept=1, renorm=True, scale=1.0):
    ids, weights = B.moe_route(raw, k, type, bias, int(sigmoid), groups, kept, renorm, scale)
    want, w, gap = R.route(x, k, bias, sigmoid, groups, kept, renorm, scale, LOWEST[type])
    top = 1.0 + (np.abs(bias).max() if bias is not None else 0.0)
    clear = gap > (2.0**-20 * 2 * top if bias is not None else 0.0)
    assert clear.mean() > 0.9
    assert np.array_equal(ids[clear], want[clear])
    assert (np.abs(weights[clear] - w[clear]) <= 2.0**-18 * np.abs(w[clear]) + 1e-37).all()
    return ids, weights


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (3, 2, 2), (5, 63, 8), (64, 64, 4), (17, 65, 1), (33, 100, 6),
                                              (9, 256, 8), (7, 257, 64), (6, 1000, 5), (4, 1024, 16)])
@pytest.mark.parametrize("sigmoid,renorm,scale", [(False, True, 1.0), (True, False, 2.5)])
def test_route(type, tokens, experts, k, sigmoid, renorm, scale):
    raw, x = stored(normal(np.random.default_rng(tokens + experts), tokens, experts, outliers=False) * 2, type)
    check_route(raw, x, type, k, sigmoid=sigmoid, renorm=renorm, scale=scale)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("experts,groups,kept,k", [(8, 2, 1, 3), (64, 8, 3, 6), (256, 8, 4, 8), (60, 4, 2, 5), (100, 50, 7, 9),
                                                   (96, 3, 3, 4), (1024, 64, 10, 8), (12, 12, 5, 5)])
@pytest.mark.parametrize("biased,sigmoid", [(False, False), (True, True), (True, False), (False, True)])
def test_route_groups_and_bias(type, experts, groups, kept, k, biased, sigmoid):
    rng = np.random.default_rng(experts * kept + k)
    raw, x = stored(normal(rng, 40, experts, outliers=False) * 1.5, type)
    bias = np.round(rng.standard_normal(experts) * 50).astype(np.float32) * np.float32(0.002) if biased else None
    check_route(raw, x, type, k, bias, sigmoid, groups, kept)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_route_masks(type, sigmoid, biased, groups, kept):
    # closed experts: -infinity, the type's lowest value, NaN; rows with fewer
    # open than chosen, with none, with all logits equal, with +infinity
    rng = np.random.default_rng(4)
    experts, k = 32, 6
    x = normal(rng, 24, experts, outliers=False)
    low = LOWEST[type]
    x[0], x[1], x[2] = -np.inf, low, np.nan
    x[3, :30], x[4, 3:], x[5, ::2], x[6, 1:] = -np.inf, low, np.nan, low
    x[7], x[8], x[9] = 0.0, -30.0, 1.25
    x[10, 5], x[11, 9], x[11, 4] = np.inf, np.inf, 2.0
    x[12] = np.where(np.arange(experts) % 3 == 0, 3.0, -np.inf)
    x[13, 8:] = -np.inf
    x[14] *= 100
    raw, x64 = stored(x, type)
    if type != B.TYPE_F32:
        x64 = np.where(np.abs(x64) > -low, np.copysign(np.inf, x64), x64)
    bias = (rng.integers(-3, 4, experts) * 0.25).astype(np.float32) if biased else None
    with np.errstate(invalid="ignore"):
        ids, weights = check_route(raw, x64, type, k, bias, sigmoid, groups, kept)
    assert (ids[:3] == -1).all() and (weights[:3] == 0).all()
    assert (np.isfinite(weights)).all()
    if not biased and groups == 1:
        assert ids[7].tolist() == list(range(k)) and ids[12].tolist() == [0, 3, 6, 9, 12, 15]
        assert ids[3].tolist()[2:] == [-1] * 4 and ids[6].tolist() == [0] + [-1] * 5


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (5, 63, 8), (33, 100, 6), (9, 256, 8), (4, 1024, 16), (7, 257, 64)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renorm,scale", [(True, 1.0), (False, 2.5)])
def test_route_backward(type, tokens, experts, k, sigmoid, renorm, scale):
    rng = np.random.default_rng(tokens + experts + k)
    x = normal(rng, tokens, experts, outliers=False)
    x[0, experts // 2:] = -np.inf
    raw, x64 = stored(x, type)
    ids, _, _ = R.route(x64, k, sigmoid=sigmoid, renorm=renorm, scale=scale)
    dw = rng.standard_normal((tokens, k)).astype(np.float32)
    got = values(B.moe_route_backward(raw, ids, dw, type, int(sigmoid), renorm, scale), type)
    want = R.route_backward(x64, ids, dw, sigmoid, renorm, scale)
    total = R.weights_of(x64, ids, sigmoid, False, 1.0).sum(1, keepdims=True)
    size = np.abs(dw).max(1, keepdims=True) * scale * (1.0 / np.maximum(total, 1e-30) if renorm else 1.0)
    scores = R.scores(x64, sigmoid)
    assert (np.abs(got - want) <= 2.0**-16 * size * scores + ROUNDING[type] * np.abs(want) + 2.0**-25).all()
    assert (got[~np.isfinite(x64)] == 0).all()


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renorm,scale", [(True, 1.0), (False, 2.5), (True, 2.5)])
def test_route_backward_is_the_derivative(sigmoid, renorm, scale):
    rng = np.random.default_rng(8)
    tokens, experts, k, h = 6, 20, 4, 1e-5
    x = normal(rng, tokens, experts, outliers=False).astype(np.float64)
    x = x.astype(np.float32).astype(np.float64)
    ids, _, _ = R.route(x, k, sigmoid=sigmoid)
    dw = rng.standard_normal((tokens, k)).astype(np.float32)
    got = B.moe_route_backward(x, ids, dw, B.TYPE_F32, int(sigmoid), renorm, scale)
    want = np.zeros_like(x)
    for e in range(experts):
        up, down = x.copy(), x.copy()
        up[:, e] += h
        down[:, e] -= h
        want[:, e] = ((R.weights_of(up, ids, sigmoid, renorm, scale) - R.weights_of(down, ids, sigmoid, renorm, scale)) * dw).sum(1) / (2 * h)
    # differences in 64 bits are good to about h^2 and 1e-16 / h
    assert (np.abs(got - want) <= 2e-5).all()


@pytest.mark.parametrize("tokens,k,experts", [(0, 1, 4), (1, 1, 1), (5, 3, 8), (64, 4, 32), (1000, 6, 100), (3000, 8, 256), (41, 2, 1024)])
def test_plan(tokens, k, experts):
    rng = np.random.default_rng(tokens + k)
    ids = rng.integers(-1, experts + 1, (tokens, k)).astype(np.int32)  # some of no expert, above and below
    if tokens > 100:
        ids[ids == 3] = 5  # one expert without pairs, one with twice as many
        ids[7] = np.array([2**31 - 1] * k, np.int32)
        ids[9] = -(2**31)
    offsets, order = B.moe_plan(ids, experts)
    want_offsets, want_order = R.plan(ids, experts)
    assert np.array_equal(offsets, want_offsets)
    assert np.array_equal(order, want_order)


def choices(rng, tokens, k, experts, skew=True):
    p = 1.0 / np.arange(1, experts + 1) if skew else np.ones(experts)
    ids = np.stack([rng.choice(experts, k, replace=False, p=p / p.sum()) for _ in range(tokens)]).astype(np.int32)
    weights = rng.random((tokens, k)).astype(np.float32)
    if tokens > 2:
        ids[1], ids[2, 0] = -1, experts + 3  # a token of no expert; an id that is none
    return ids, weights


@pytest.mark.parametrize("type,out", [(B.TYPE_F32, B.TYPE_F32), (B.TYPE_BF16, B.TYPE_BF16), (B.TYPE_F16, B.TYPE_F32)])
@pytest.mark.parametrize("tokens,k,experts,inputs,n", [(1, 1, 1, 1, 1), (1, 2, 4, 300, 130), (3, 3, 70, 257, 33),
                                                       (16, 4, 8, 512, 200), (70, 2, 5, 130, 257), (300, 1, 3, 96, 64),
                                                       (200, 4, 16, 700, 129)])
def test_layer(type, out, tokens, k, experts, inputs, n):
    rng = np.random.default_rng(tokens + experts * inputs)
    raw, x = stored(normal(rng, tokens, inputs), type)
    wraw, w = stored(normal(rng, experts, n, inputs), type)
    draw, dy = stored(normal(rng, tokens, n) * 1e-2, type)
    ids, weights = choices(rng, tokens, k, experts)
    wr, wt = B.mx4_encode(wraw, type, columns=True)
    layer = B.MoeLinear(wr, wt)
    got = values(layer.forward(raw, ids, weights, type, out), out)
    y, want, dx, dweights, dw = R.experts_layer(x, ids, weights, w, dy)
    offsets, order = R.plan(ids, experts)
    assert np.array_equal(layer.offsets.download(np.int32, experts + 1), offsets)
    assert np.array_equal(layer.order.download(np.int32, tokens * k), order)
    # a sum's bound, from the magnitudes of its factors
    xa, wa = np.abs(R.rounded(x)), np.stack([np.abs(R.rounded(w[e])) for e in range(experts)])
    da, wta = np.abs(R.rounded(dy)), np.stack([np.abs(R.rounded(np.ascontiguousarray(w[e].T))) for e in range(experts)])
    real = (ids >= 0) & (ids < experts)
    at = np.where(real, ids, 0)
    ya = np.einsum("ti,tjni->tjn", xa, wa[at]) * real[..., None]
    za = np.einsum("tn,tjin->tji", da, wta[at]) * real[..., None]
    got_y = layer.y.download(np.float32, tokens * k * n).reshape(tokens, k, n)
    assert (np.abs(got_y - y) <= inputs * 2.0**-23 * ya + 2.0**-24 * np.abs(y)).all()
    wy = weights[..., None] * ya
    assert (np.abs(got - want) <= (inputs + k) * 2.0**-23 * wy.sum(1) + ROUNDING[out] * np.abs(want) + 1e-30).all()
    gx, gweights, gw = layer.backward(draw, type, out)
    # z is held in the gradients' type before the join
    wz = weights[..., None] * za
    assert (np.abs(values(gx, out) - dx) <= ((n + k) * 2.0**-23 + ROUNDING[out]) * wz.sum(1) + ROUNDING[out] * np.abs(dx) + 1e-30).all()
    assert (np.abs(gweights - dweights) <= (inputs + n) * 2.0**-23 * (ya * np.abs(dy)[:, None]).sum(2) + 1e-30).all()
    assert (gweights[~real] == 0).all()
    gw = values(gw, out)
    for e in range(experts):
        t, j = np.nonzero(ids == e)
        g = np.abs(weights[t, j, None] * dy[t]).astype(np.float64)
        bound = 2 * (len(t) + 1) * 2.0**-23 * (np.abs(R.rounded(np.ascontiguousarray(g.T))) @ np.abs(R.rounded(np.ascontiguousarray(x[t].T))).T) if len(t) else 0.0
        assert (np.abs(gw[e] - dw[e]) <= bound + ROUNDING[out] * np.abs(dw[e]) + 1e-30).all()


@pytest.mark.parametrize("tokens,k,experts,inputs,n", [(1500, 2, 4, 300, 520), (3000, 2, 3, 256, 1400), (2600, 4, 40, 130, 300),
                                                       (2000, 2, 64, 130, 200), (1500, 4, 150, 130, 260)])
def test_layer_in_large_tiles(tokens, k, experts, inputs, n):
    # integers whose sums are exact: the forward pass, the gradient of x and the
    # weights' own, element by element
    rng = np.random.default_rng(tokens)

    def of(*shape):
        a = rng.integers(-2, 3, shape).astype(np.float32)
        a[..., ::32] = 4.0
        return a

    x, w, dy = of(tokens, inputs), of(experts, n, inputs), of(tokens, n)
    w[:, ::32], dy[::1, ::32] = 4.0, 4.0
    ids, _ = choices(rng, tokens, k, experts)
    weights = rng.choice([0.5, 1.0, 2.0], (tokens, k)).astype(np.float32)
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    got = layer.forward(x, ids, weights)
    gx, gweights, gw = layer.backward(dy)
    y, z = np.zeros((tokens, k, n)), np.zeros((tokens, k, inputs))
    for e in range(experts):
        t, j = np.nonzero(ids == e)
        y[t, j] = x[t] @ w[e].T
        z[t, j] = dy[t] @ w[e]
        g = (weights[t, j, None] * dy[t]).astype(np.float64)
        if len(t):
            want = R.rounded(np.ascontiguousarray(g.T)) @ R.rounded(np.ascontiguousarray(x[t].T.astype(np.float64))).T
            assert np.array_equal(gw[e], want.astype(np.float32)), e
        else:
            assert (gw[e] == 0).all()
    real = (ids >= 0) & (ids < experts)
    wt = np.where(real, weights, 0.0)[..., None]
    assert np.array_equal(got, (y * wt).sum(1).astype(np.float32))
    assert np.array_equal(gx, (z * wt).sum(1).astype(np.float32))
    assert (np.abs(gweights - (y * dy[:, None]).sum(2)) <= n * 2.0**-23 * (np.abs(y) * np.abs(dy[:, None])).sum(2)).all()


def test_layer_types_and_parts_of_the_backward_pass():
    # gradients of another type than the inputs, and each gradient asked for by
    # itself, give what the whole call gives on the same values
    rng = np.random.default_rng(77)
    tokens, k, experts, inputs, n = 90, 2, 5, 140, 75
    x, w = B.to_bf16(normal(rng, tokens, inputs)), normal(rng, experts, n, inputs)
    dy16 = B.to_bf16(normal(rng, tokens, n) * 0.01)
    dy32 = B.from_bf16(dy16)
    ids, weights = choices(rng, tokens, k, experts)
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    layer.forward(x, ids, weights, B.TYPE_BF16)
    whole = layer.backward(dy16, B.TYPE_BF16)
    for got, want in zip(layer.backward(dy32, B.TYPE_F32), whole):
        assert np.array_equal(got, want)
    L, d = B.lib(), B.DeviceBuffer.from_array(dy16)
    work = B.DeviceBuffer(L.bsq_moe_linear_backward_workspace(tokens, k, n, inputs, experts))
    outs = [B.DeviceBuffer(v.nbytes) for v in whole]
    for only in range(3):
        dx, dweights, dw = (outs[i].ptr if i == only else None for i in range(3))
        B.check(L.bsq_moe_linear_backward(d.ptr, B.TYPE_BF16, tokens, n, n, layer.x.ptr, B.TYPE_BF16, inputs, inputs,
                                          layer.ids.ptr, layer.weights.ptr, k, layer.offsets.ptr, layer.order.ptr,
                                          layer.y.ptr, 0, layer.wt.codes.ptr, layer.wt.scales.ptr, experts, dx, inputs,
                                          dweights, dw, 0, work.ptr, work.nbytes, None), "backward")
        B.check(L.bsq_stream_synchronize(None), "sync")
        got = outs[only].download(np.float32, whole[only].size).reshape(whole[only].shape)
        assert np.array_equal(got, whole[only]), only


def test_layer_of_no_tokens():
    layer = B.MoeLinear(*B.mx4_encode(np.ones((3, 40, 50), np.float32), columns=True))
    out = layer.forward(np.zeros((0, 50), np.float32), np.zeros((0, 2), np.int32), np.zeros((0, 2), np.float32))
    assert out.shape == (0, 40)
    dx, dweights, dw = layer.backward(np.zeros((0, 40), np.float32))
    assert dx.size == 0 and dweights.size == 0 and (dw == 0).all()


@pytest.mark.parametrize("bits", [B.TYPE_F32, B.TYPE_BF16])
def test_layer_all_tokens_to_one_expert_and_none(bits):
    rng = np.random.default_rng(21)
    tokens, experts, inputs, n = 150, 6, 64, 40
    x, w = normal(rng, tokens, inputs), normal(rng, experts, n, inputs)
    weights = np.ones((tokens, 1), np.float32)
    for e in (0, 5, -1):
        layer = B.MoeLinear(B.mx4_encode(w))
        got = values(layer.forward(x, np.full((tokens, 1), e, np.int32), weights, y_type=bits), B.TYPE_F32)
        if e < 0:
            assert (got == 0).all()
            continue
        a, b = R.rounded(x.astype(np.float64)), R.rounded(w[e].astype(np.float64))
        assert (np.abs(got - a @ b.T) <= R.product_bound(a, b, ROUNDING[bits] + 2.0**-24)).all()


def test_route_then_layer():
    # as a model runs them: the router's ids and weights go to the layer, the
    # layer's gradient of the weights back through the router
    rng = np.random.default_rng(31)
    tokens, experts, k, inputs, n = 50, 12, 3, 96, 80
    x, w = normal(rng, tokens, inputs), normal(rng, experts, n, inputs)
    logits, dy = normal(rng, tokens, experts), normal(rng, tokens, n)
    ids, weights = B.moe_route(logits, k)
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    out = layer.forward(x, ids, weights)
    _, dweights, _ = layer.backward(dy)
    dlogits = B.moe_route_backward(logits, ids, dweights)
    y, want, _, want_dweights, _ = R.experts_layer(x.astype(np.float64), ids, weights, w.astype(np.float64), dy.astype(np.float64))
    assert np.linalg.norm(out - want) <= 1e-5 * np.linalg.norm(want)
    d = R.route_backward(logits.astype(np.float64), ids, want_dweights, False, True, 1.0)
    assert np.linalg.norm(dlogits - d) <= 1e-5 * np.linalg.norm(d)
