"""MX4 encode, decode, products and the dense layer (csrc/mx4.hip,
csrc/mx4_gemm.hip) against their definitions in 64 bits (_mx4ref.py).

Codes, scales and decoded values are defined bit by bit.  Products are held to
the worst case of K additions in FP32 (product_bound) plus the rounding of the
output type, half a unit in the last place of 24, 8 and 11 bits: 2^-24 of a value
for FP32, 2^-8 for BF16, 2^-11 for FP16."""
import ctypes

import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B

pytestmark = pytest.mark.gpu

TYPES = [B.TYPE_F32, B.TYPE_BF16, B.TYPE_F16]
ROUNDING = {B.TYPE_F32: 2.0**-24, B.TYPE_BF16: 2.0**-8, B.TYPE_F16: 2.0**-11}


def stored(x, type):
    """(what the call takes, its values in 64 bits)."""
    if type == B.TYPE_BF16:
        b = B.to_bf16(x)
        return b, B.from_bf16(b).astype(np.float64)
    h = np.ascontiguousarray(x, np.float16 if type == B.TYPE_F16 else np.float32)
    return h, h.astype(np.float64)


def values(out, type):
    return B.from_bf16(out).astype(np.float64) if type == B.TYPE_BF16 else out.astype(np.float64)


def normal(rng, *shape, outliers=True):
    x = rng.standard_normal(shape).astype(np.float32)
    if outliers and shape[-1] > 4:
        x[..., rng.integers(0, shape[-1], max(1, shape[-1] // 200))] *= 30.0
    return x


def same(packed, x):
    codes, scales = packed.download()
    want_codes, want_scales = R.packed(x)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 255), (4, 256), (7, 257), (33, 640), (129, 130),
                                       (300, 1003)])
def test_encode_rows_and_columns(type, rows, cols):
    raw, x = stored(normal(np.random.default_rng(rows * 1000 + cols), rows, cols), type)
    r, c = B.mx4_encode(raw, type, columns=True)
    same(r, x)
    same(c, np.ascontiguousarray(x.T))
    same(B.mx4_encode(raw, type), x)  # the rows alone: another kernel
    same(B.mx4_encode(raw, type, rows=False, columns=True), np.ascontiguousarray(x.T))
    assert np.array_equal(r.decode(), R.rounded(x).astype(np.float32))


def every_value(type):
    """Every 16-bit pattern that is finite; for FP32 every tie of every scale and its
    neighbours, subnormals and the largest."""
    if type != B.TYPE_F32:
        bits = np.arange(1 << 16, dtype=np.uint16)
        v = B.from_bf16(bits) if type == B.TYPE_BF16 else bits.view(np.float16).astype(np.float32)
        return v[np.isfinite(v)]
    e = np.ldexp(np.float32(1), np.arange(-149, 128)).astype(np.float32)
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 1.5, 3, 6], np.float32)
    with np.errstate(over="ignore"):
        v = (e[:, None] * mid).ravel()
    v = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(0))])
    v = v[np.isfinite(v)]
    return np.concatenate([v, -v])


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("top", [1.0, 1.5, 6.0, 5.99, 0.011, 40000.0, 2.0**-100, 2.0**-130, 1e-38, 3e38])
def test_encode_every_value_under_a_scale(type, top):
    # blocks of one value `top` and 31 others no larger: ties and their
    # neighbours under the scale that `top` gives
    t = stored(np.array([top], np.float32), type)[1][0]
    if not np.isfinite(t):
        pytest.skip("not a value of the type")
    v = every_value(type)
    v = v[np.abs(v) <= t]
    v = v[: v.size // 31 * 31].reshape(-1, 31)
    if v.size == 0:
        pytest.skip("no smaller value")
    x = np.concatenate([np.full((len(v), 1), t, np.float32), v.astype(np.float32)], 1)
    x = np.concatenate([x, np.zeros((-len(x) % 8, 32), np.float32)]).reshape(-1, 256)
    raw, x64 = stored(x, type)
    r, c = B.mx4_encode(raw, type, columns=True)
    same(r, x64)
    same(c, np.ascontiguousarray(x64.T))


@pytest.mark.parametrize("type", TYPES)
def test_encode_block_maxima(type):
    # every magnitude as a block's largest
    v = np.abs(every_value(type))
    x = np.zeros((v.size, 32), np.float32)
    x[:, 5], x[:, 17] = v, -v / 2
    x = np.concatenate([x, np.zeros((-len(x) % 8, 32), np.float32)]).reshape(-1, 256)
    raw, x64 = stored(x, type)
    same(B.mx4_encode(raw, type), x64)


@pytest.mark.parametrize("type", TYPES)
def test_encode_not_finite(type):
    # a block with a NaN or an infinity is NaN; its neighbours are not touched
    x = normal(np.random.default_rng(5), 64, 512)
    x[3, 40], x[9, 100], x[63, 511], x[0, 0] = np.nan, np.inf, -np.inf, -np.nan
    raw, x64 = stored(x, type)
    r, c = B.mx4_encode(raw, type, columns=True)
    same(r, x64)
    same(c, np.ascontiguousarray(x64.T))
    got, want = r.decode(), R.rounded(x64)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got).sum() == 4 * 32
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)].astype(np.float32))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("shift,ld", [(0, 333), (1, 333), (3, 336), (0, 640)])
def test_encode_strides_and_alignment(type, shift, ld):
    rows, cols, batch = 70, 300, 3
    rng = np.random.default_rng(shift + ld)
    stride = rows * ld + 11
    raw, x64 = stored(normal(rng, batch * stride + shift), type)
    d = B.DeviceBuffer.from_array(raw)
    r, c = B.Mx4(rows, cols, batch), B.Mx4(cols, rows, batch)
    src = ctypes.c_void_p(d.ptr.value + shift * raw.itemsize)
    B.check(B.lib().bsq_mx4_encode(src, type, batch, rows, cols, ld, stride, r.codes.ptr, r.scales.ptr, c.codes.ptr,
                                   c.scales.ptr, None), "encode")
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    x = np.stack([np.lib.stride_tricks.as_strided(x64[shift + b * stride:], (rows, cols), (8 * ld, 8)) for b in range(batch)])
    same(r, x.reshape(-1, cols))
    same(c, np.ascontiguousarray(x.transpose(0, 2, 1)).reshape(-1, rows))


@pytest.mark.parametrize("type", TYPES)
def test_decode_every_code_and_scale(type):
    # one block for each scale byte, all sixteen codes in it; a row ld apart,
    # its end not a multiple of eight
    rows, cols, ld = 256, 37, 41
    codes = np.zeros((rows, 128), np.uint8)
    codes[:, :16] = np.tile(np.arange(16, dtype=np.uint8) | ((15 - np.arange(16, dtype=np.uint8)) << 4), (rows, 1))
    scales = np.ones((rows, 8), np.uint8) * 127
    scales[:, 0] = np.arange(256)
    dc, ds = B.DeviceBuffer.from_array(codes), B.DeviceBuffer.from_array(scales)
    size = 4 if type == B.TYPE_F32 else 2
    out = B.DeviceBuffer.from_array(np.full(rows * ld * size, 0x5A, np.uint8))
    B.check(B.lib().bsq_mx4_decode(dc.ptr, ds.ptr, rows, cols, out.ptr, type, ld, None), "decode")
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    t = {B.TYPE_F32: np.float32, B.TYPE_BF16: np.uint16, B.TYPE_F16: np.float16}[type]
    got = out.download(t, rows * ld).reshape(rows, ld)
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(rows, 256)
    with np.errstate(over="ignore"):
        want = R.decode(nibbles, scales, cols)
        want = B.to_bf16(want.astype(np.float32)) if type == B.TYPE_BF16 else want.astype(t)
    if type == B.TYPE_BF16:
        nan = scales[:, 0] == 255
        assert np.array_equal(got[~nan, :cols], want[~nan])
        assert np.isnan(B.from_bf16(got[nan, :32])).all()
    else:
        assert np.array_equal(got[:, :cols], want, equal_nan=True)
    assert (np.ascontiguousarray(got[:, cols:]).view(np.uint8) == 0x5A).all()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 129, 32), (2, 64, 257), (3, 1, 1000), (5, 300, 4096), (16, 128, 256),
                                   (17, 31, 513), (33, 257, 2048), (64, 64, 12000), (100, 1000, 96), (128, 128, 128),
                                   (129, 127, 300), (255, 600, 1500), (300, 257, 768), (513, 514, 515)])
def test_product(out, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    x, w = normal(rng, m, k), normal(rng, n, k)
    a, b = B.mx4_encode(x), B.mx4_encode(w)
    aq, bq = R.rounded(x.astype(np.float64)), R.rounded(w.astype(np.float64))
    got = values(B.mx4_product(a, b, out), out)
    want = aq @ bq.T
    bound = R.product_bound(aq, bq, ROUNDING[out])
    if out == B.TYPE_F16:
        bound = bound + 2.0**-25  # subnormal steps
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


@pytest.mark.parametrize("m,n,k", [(600, 600, 200), (400, 500, 1800), (900, 700, 3000), (2100, 1000, 513), (2100, 1000, 256),
                                   (2300, 2000, 300), (2300, 2000, 1100), (2950, 2948, 256), (2950, 2948, 900),
                                   (5000, 1800, 2049), (120, 70, 20000), (130, 300, 9000)])
def test_product_of_every_cut(m, n, k):
    # the tiles and teams that these sizes take on 256 CUs: 64 alone, in twos and
    # fours, 128 alone and in twos, 256; odd and even slices; split shared axes.
    # Every element against a sum over integers that is exact in FP32.
    rng = np.random.default_rng(m + n + k)
    x = rng.integers(-2, 3, (m, k)).astype(np.float32)
    w = rng.integers(-2, 3, (n, k)).astype(np.float32)
    x[:, ::32], w[:, ::32] = 4.0, 4.0  # scale 1 in every block
    want = x @ w.T  # below 2^24: exact
    a, b = B.mx4_encode(x), B.mx4_encode(w)
    assert np.array_equal(B.mx4_product(a, b), want)
    assert np.array_equal(B.mx4_product(a, b, B.TYPE_BF16), B.to_bf16(want))


def test_product_is_exact_where_sums_are():
    # integers: every partial sum is exact in FP32, so the result is too, in any
    # order, and a misplaced block or scale shows
    rng = np.random.default_rng(2)
    for m, n, k in ((1, 300, 1024), (7, 513, 2304), (40, 200, 768), (260, 390, 1280)):
        x = rng.choice(R.LEVELS, (m, k)) * rng.choice([-1, 1], (m, k)) * 2.0 ** rng.integers(0, 4, (m, k // 32)).repeat(32, 1)
        w = rng.choice(R.LEVELS, (n, k)) * rng.choice([-1, 1], (n, k)) * 2.0 ** rng.integers(0, 4, (n, k // 32)).repeat(32, 1)
        x[:, ::32], w[:, ::32] = 6.0 * np.sign(x[:, ::32] + 0.1) * 8, 6.0 * np.sign(w[:, ::32] + 0.1) * 8  # the blocks' scale is 8
        xq, wq = R.rounded(x), R.rounded(w)
        assert np.array_equal(B.mx4_product(B.mx4_encode(x), B.mx4_encode(w)), (xq @ wq.T).astype(np.float32))
        assert np.array_equal(B.mx4_linear(x, B.mx4_encode(w)), (xq @ wq.T).astype(np.float32))


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_product_not_finite(m):
    # a NaN or infinity makes its own row (or column) NaN and no other
    rng = np.random.default_rng(m)
    x, w = normal(rng, m, 700), normal(rng, 150, 700)
    x[m // 2, 333], w[7, 12], w[149, 699] = np.inf, np.nan, -np.inf
    got = B.mx4_product(B.mx4_encode(x), B.mx4_encode(w))
    want = np.zeros((m, 150), bool)
    want[m // 2], want[:, 7], want[:, 149] = True, True, True
    assert np.array_equal(np.isnan(got), want)


@pytest.mark.parametrize("m,n,k", [(1, 200, 300), (40, 200, 300), (300, 200, 300)])
def test_product_extreme_scales(m, n, k):
    # scales near both ends of their range: 2^-126 and 2^126
    rng = np.random.default_rng(k)
    x = normal(rng, m, k).astype(np.float64)
    w = normal(rng, n, k).astype(np.float64)
    for sx, sw in ((2.0**100, 2.0**-110), (2.0**-120, 2.0**118), (2.0**50, 2.0**40)):
        a, b = (x * sx).astype(np.float32), (w * sw).astype(np.float32)
        aq, bq = R.rounded(a.astype(np.float64)), R.rounded(b.astype(np.float64))
        got = B.mx4_product(B.mx4_encode(a), B.mx4_encode(b)).astype(np.float64)
        assert (np.abs(got - aq @ bq.T) <= R.product_bound(aq, bq, 2.0**-24)).all()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (4, 64, 5000), (16, 700, 520), (31, 33, 257), (64, 1024, 2048),
                                   (200, 300, 700)])
def test_linear_is_encode_and_product(type, m, n, k):
    rng = np.random.default_rng(m + n + k)
    raw, x = stored(normal(rng, m, k), type)
    w = B.mx4_encode(normal(rng, n, k))
    y, xt = B.mx4_linear(raw, w, type, keep=True)
    same(xt, np.ascontiguousarray(x.T))
    # the same sums whether the transpose is kept or not
    assert np.array_equal(y, B.mx4_linear(raw, w, type))
    aq, bq = R.rounded(x), w.decode().astype(np.float64)
    assert (np.abs(y - aq @ bq.T) <= R.product_bound(aq, bq, 2.0**-24)).all()


def test_linear_strides():
    m, n, k, ldx, ldo = 9, 70, 300, 307, 81
    rng = np.random.default_rng(9)
    x = normal(rng, m, ldx)
    w = B.mx4_encode(normal(rng, n, k))
    d, out = B.DeviceBuffer.from_array(x), B.DeviceBuffer.from_array(np.full(m * ldo, 7.0, np.float32))
    work = B.DeviceBuffer(B.lib().bsq_mx4_linear_workspace(m, n, k))
    B.check(B.lib().bsq_mx4_linear(d.ptr, 0, m, k, ldx, w.codes.ptr, w.scales.ptr, n, out.ptr, 0, ldo, None, None, work.ptr,
                                   work.nbytes, None), "linear")
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    got = out.download(np.float32, m * ldo).reshape(m, ldo)
    assert np.array_equal(got[:, :n], B.mx4_linear(np.ascontiguousarray(x[:, :k]), w))
    assert (got[:, n:] == 7.0).all()


@pytest.mark.parametrize("type,g", [(B.TYPE_F32, B.TYPE_F32), (B.TYPE_BF16, B.TYPE_BF16), (B.TYPE_BF16, B.TYPE_F32)])
@pytest.mark.parametrize("m,n,k", [(1, 5, 7), (33, 70, 129), (256, 300, 200), (400, 130, 517)])
def test_linear_backward(type, g, m, n, k):
    rng = np.random.default_rng(m * n + k)
    raw, x = stored(normal(rng, m, k), type)
    wraw, w = stored(normal(rng, n, k), type)
    draw, dy = stored(normal(rng, m, n) * 1e-3, type)
    wr, wt = B.mx4_encode(wraw, type, columns=True)
    _, xt = B.mx4_linear(raw, wr, type, keep=True)
    dx, dw = B.mx4_linear_backward(draw, xt, wt, type, g)
    t = np.ascontiguousarray
    for got, a, b in ((dx, R.rounded(dy), R.rounded(t(w.T))), (dw, R.rounded(t(dy.T)), R.rounded(t(x.T)))):
        assert (np.abs(values(got, g) - a @ b.T) <= R.product_bound(a, b, ROUNDING[g])).all()


def test_linear_backward_is_the_derivative():
    # values of the format whose neighbours are too, so that rounding moves
    # nothing: L = <dy, out> is linear in x and in w, and its differences are
    # exactly the gradients
    rng = np.random.default_rng(11)
    m, n, k = 6, 10, 40

    def of(*shape):
        return rng.choice([-1.0, -0.5, 0.5, 1.0], shape)

    x, w, dy = of(m, k), of(n, k), of(m, n)
    # both ways' blocks hold a 4, so that every scale is 1 and holds steps of a half
    for a in (x, w, dy):
        a[0, :], a[:, 0] = 4.0, 4.0
        a[32:, :][:1] = 4.0
        a[:, 32:][:, :1] = 4.0

    def loss(x, w):
        return float((dy * B.mx4_linear(x, B.mx4_encode(w)).astype(np.float64)).sum())

    wr, wt = B.mx4_encode(w, columns=True)
    _, xt = B.mx4_linear(x, wr, keep=True)
    dx, dw = B.mx4_linear_backward(dy, xt, wt)
    for a, d, at in ((x, dx, (3, 17)), (x, dx, (5, 39)), (w, dw, (2, 3)), (w, dw, (9, 35))):
        up = a.copy()
        up[at] += 0.5
        diff = (loss(up, w) - loss(x, w)) if a is x else (loss(x, up) - loss(x, w))
        assert diff == 0.5 * d[at], (at, diff, d[at])


class Hip:
    """The HIP runtime that the library runs on, for a stream and a graph of the
    caller's own."""

    def __init__(self):
        B.lib()
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64.so" in line)
        self.hip = ctypes.CDLL(path)

    def __call__(self, name, *args):
        rc = getattr(self.hip, name)(*args)
        assert rc == 0, (name, rc)


def test_other_stream_and_replays():
    # work on a stream of the caller's, captured once and replayed with new
    # inputs, eager calls between the replays
    L, hip, stream = B.lib(), Hip(), ctypes.c_void_p()
    hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)  # does not wait for the null stream
    m, n, k, experts, chosen = 24, 640, 1536, 4, 2
    rng = np.random.default_rng(3)
    w = B.mx4_encode(normal(rng, experts, n, k))
    x, work = B.DeviceBuffer(m * k * 4), B.DeviceBuffer(max(L.bsq_mx4_linear_workspace(m, n, k),
                                                           L.bsq_moe_linear_workspace(m, chosen, n, k, experts)))
    logits, ids, weights = B.DeviceBuffer(m * experts * 4), B.DeviceBuffer(m * chosen * 4), B.DeviceBuffer(m * chosen * 4)
    offsets, order, y = B.DeviceBuffer(4 * experts + 4), B.DeviceBuffer(m * chosen * 4), B.DeviceBuffer(m * chosen * n * 4)
    outs = [B.DeviceBuffer(m * n * 4) for _ in range(2)]

    def step():
        B.check(L.bsq_mx4_linear(x.ptr, 0, m, k, k, w.codes.ptr, w.scales.ptr, n, outs[0].ptr, 0, n, None, None, work.ptr,
                                 work.nbytes, stream), "linear")
        B.check(L.bsq_moe_route(logits.ptr, 0, m, experts, experts, None, 0, 1, 1, chosen, 1, 1.0, ids.ptr, weights.ptr,
                                stream), "route")
        B.check(L.bsq_moe_linear(x.ptr, 0, m, k, k, ids.ptr, weights.ptr, chosen, w.codes.ptr, w.scales.ptr, experts, n,
                                 offsets.ptr, order.ptr, y.ptr, 0, outs[1].ptr, 0, n, work.ptr, work.nbytes, stream), "layer")

    def inputs():
        a, b = normal(rng, m, k), normal(rng, m, experts)
        x.upload(a)
        logits.upload(b)
        return a

    def results():
        hip("hipStreamSynchronize", stream)
        got = [o.download(np.float32, m * n).copy() for o in outs]
        for o in outs:
            o.zero()
        hip("hipDeviceSynchronize")
        return got

    inputs()
    step()
    results()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, 2)
    step()
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    for _ in range(3):
        a = inputs()
        step()
        want = results()
        hip("hipGraphLaunch", run, stream)
        got = results()
        assert all(np.array_equal(g, v) for g, v in zip(got, want))
    xq, wq = R.rounded(a.astype(np.float64)), w.decode()[:n].astype(np.float64)
    assert (np.abs(got[0].reshape(m, n) - xq @ wq.T) <= R.product_bound(xq, wq, 2.0**-24)).all()
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", stream)
