"""Calls of more threads than 32 bits count, past which a launch is cut without
an error (csrc/mx4.hip, mx4_gemm.hip, moe.hip): those that go by tiles are
refused before anything is queued, those that go by tokens or pairs run, and
experts without pairs take no tiles."""
import ctypes

import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B
from test_mx4_refusals import D, refused


def test_tiles_past_a_launch_are_refused():
    # without a GPU: a call that queued something first would fail with the
    # runtime's own error
    L = B.lib()
    refused(L.bsq_mx4_encode(D, 0, (1 << 21) + 1, 1, 1, 1, 1, D, D, D, D, None), "too large")
    refused(L.bsq_mx4_encode(D, 1, (1 << 22) + 1, 1, 1, 1, 1, D, D, D, D, None), "too large")
    n = (1 << 31) - 1
    refused(L.bsq_mx4_product(D, D, 1, D, D, n, 256, D, 0, n, None, 0, None), "product: too large")
    refused(L.bsq_mx4_linear(D, 0, 1, 256, 256, D, D, n, D, 0, n, None, None, D, 1 << 50, None), "product: too large")
    n = 1 << 22
    refused(L.bsq_moe_linear(D, 0, 1024, 64, 64, D, D, 1, D, D, 256, n, D, D, D, 0, D, 0, n, D, 1 << 60, None), "product: too large")
    refused(L.bsq_moe_linear_backward(D, 0, 1024, 64, 64, D, 0, n, n, D, D, 1, D, D, D, 0, D, D, 256, D, n, None, None, 0, D,
                                      1 << 60, None), "product: too large")


def memory(*sizes):
    try:
        return [B.DeviceBuffer(s) for s in sizes]
    except B.BsqError:
        pytest.skip(f"needs {sum(sizes) / 1e9:.0f} GB of device memory")


def at(buffer, offset):
    return ctypes.c_void_p(buffer.ptr.value + offset)


MANY = (1 << 26) + 5  # a wave each: 2^32 + 320 threads


def tiled(one, count):
    """`count` rows of a pattern, uploaded; its period is prime."""
    reps = -(-count // len(one))
    return B.DeviceBuffer.from_array(np.tile(one, (reps,) + (1,) * (one.ndim - 1))[:count])


def same_throughout(buffer, one, count, equal):
    got = buffer.download(one.dtype, count * one[0].size).reshape(count, -1)
    for i in range(0, count, len(one)):
        part = got[i: i + len(one)]
        assert equal(part, one.reshape(len(one), -1)[: len(part)]), i


@pytest.mark.gpu
def test_routing_and_its_gradient_of_many_tokens():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1000003, 2)).astype(np.float32)
    ids, weights, dw, dx = memory(4 * MANY, 4 * MANY, 4 * MANY, 8 * MANY)
    logits, L = tiled(x, MANY), B.lib()
    B.check(L.bsq_moe_route(logits.ptr, 0, MANY, 2, 2, None, 0, 1, 1, 1, 0, 1.0, ids.ptr, weights.ptr, None), "route")
    B.check(L.bsq_stream_synchronize(None), "sync")
    best = x.argmax(1).astype(np.int32)
    same_throughout(ids, best, MANY, np.array_equal)
    s = R.scores(x, False)
    want = s.max(1).astype(np.float32)
    same_throughout(weights, want, MANY, lambda a, b: np.allclose(a, b, rtol=2.0**-18, atol=0))
    dw.upload(np.ones(MANY, np.float32))
    dx.zero()
    B.check(L.bsq_moe_route_backward(logits.ptr, 0, MANY, 2, 2, 0, 1, 0, 1.0, ids.ptr, dw.ptr, dx.ptr, 2, None), "backward")
    B.check(L.bsq_stream_synchronize(None), "sync")
    want = R.route_backward(x, best[:, None], np.ones((len(x), 1)), False, False, 1.0).astype(np.float32)
    same_throughout(dx, want, MANY, lambda a, b: (np.abs(a - b) <= 2.0**-16).all())


@pytest.mark.gpu
def test_gradient_of_the_routing_weights_of_many_pairs():
    rng = np.random.default_rng(2)
    y, dy = (rng.standard_normal(1000003).astype(np.float32) for _ in range(2))
    L = B.lib()
    need = B.workspace("bsq_moe_linear_backward_workspace", MANY, 1, 1, 1, 1)
    work, ids, dweights, other = memory(need, 4 * MANY, 4 * MANY, 4 * MANY)
    ids.zero()
    dy_, y_ = tiled(dy, MANY), tiled(y, MANY)
    B.check(L.bsq_moe_linear_backward(dy_.ptr, 0, MANY, 1, 1, None, 0, 1, 0, ids.ptr, other.ptr, 1, other.ptr, other.ptr,
                                      y_.ptr, 0, None, None, 1, None, 0, dweights.ptr, None, 0, work.ptr, work.nbytes, None),
            "backward")
    B.check(L.bsq_stream_synchronize(None), "sync")
    same_throughout(dweights, y * dy, MANY, np.array_equal)


@pytest.mark.gpu
def test_join_of_many_pieces():
    # three pieces of eight columns a token, 2^32 + 2 in all: all rows alike but
    # for some around the ends of the launches' turns
    tokens, n = 1431655766, 17
    y, out, ids, weights = memory(2 * n * tokens, 2 * n * tokens, 4 * tokens, 4 * tokens)
    L = B.lib()
    B.check(L.bsq_device_memset(y.ptr, 0x3F, y.nbytes), "memset")        # BF16 0.74609375
    B.check(L.bsq_device_memset(weights.ptr, 0x40, weights.nbytes), "memset")  # 3.00392...
    ids.zero()
    out.zero()
    some = sorted({0, 1, tokens - 1, tokens - 2, *((i << 28) // 3 + d for i in range(1, 16) for d in (-1, 0, 1))})
    rng = np.random.default_rng(3)
    rows = {t: B.to_bf16(rng.standard_normal(n).astype(np.float32)) for t in some}
    for t, r in rows.items():
        B.check(L.bsq_memcpy_h2d(at(y, 2 * n * t), r.ctypes.data, r.nbytes), "H2D")
    B.check(L.bsq_moe_combine(y.ptr, B.TYPE_BF16, tokens, 1, n, ids.ptr, weights.ptr, 1, out.ptr, B.TYPE_BF16, n, None), "combine")
    B.check(L.bsq_stream_synchronize(None), "sync")
    w = np.frombuffer(b"\x40" * 4, np.float32)[0]
    plain = np.full(n, 0x3F3F, np.uint16)
    for t in some + rng.integers(0, tokens, 500).tolist():
        got = np.empty(n, np.uint16)
        B.check(L.bsq_memcpy_d2h(got.ctypes.data, at(out, 2 * n * t), got.nbytes), "D2H")
        assert np.array_equal(got, B.to_bf16(w * B.from_bf16(rows.get(t, plain)))), t


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,k,experts,inputs,n", [(1, 4, 256, 300, 70), (1, 1, 1024, 64, 40), (8, 4, 1024, 96, 33),
                                                       (3, 64, 256, 64, 20), (5, 2, 200, 2600, 17)])
def test_few_tokens_and_many_experts(tokens, k, experts, inputs, n):
    # a launch has as many row tiles as there can be; sums are exact
    rng = np.random.default_rng(experts + tokens)
    x, w, dy = (rng.integers(-2, 3, s).astype(np.float32) for s in ((tokens, inputs), (experts, n, inputs), (tokens, n)))
    x[:, ::32], w[:, :, ::32], w[:, ::32], dy[:, ::32] = 4.0, 4.0, 4.0, 4.0
    ids = np.stack([rng.choice(experts, k, replace=False) for _ in range(tokens)]).astype(np.int32)
    ids[0, 0] = experts - 1
    if k > 2:
        ids[-1, 1] = -1
    weights = rng.choice([0.5, 1.0, 2.0], (tokens, k)).astype(np.float32)
    layer = B.MoeLinear(*B.mx4_encode(w, columns=True))
    got = layer.forward(x, ids, weights)
    dx, _, _ = layer.backward(dy)
    real = np.where(ids >= 0, weights, 0.0)
    picked = w[np.maximum(ids, 0)].astype(np.float64)
    assert np.array_equal(got, np.einsum("tk,tkni,ti->tn", real, picked, x).astype(np.float32))
    assert np.array_equal(dx, np.einsum("tk,tkni,tn->ti", real, picked, dy).astype(np.float32))
