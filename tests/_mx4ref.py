"""The MX4 format and its layers from their definitions, in numpy and 64 bits:
what the GPU operators are compared with."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SLICE = 256


def pad(x, multiple):
    extra = -x.shape[-1] % multiple
    return np.concatenate([x, np.zeros((*x.shape[:-1], extra), x.dtype)], -1) if extra else x


def encode(x):
    """(codes 0..15, scale bytes) of float64 x along its last axis, padded to a slice."""
    b = pad(np.asarray(x, np.float64), SLICE).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    b = np.where(bad, 0.0, b)
    m, e = np.frexp(np.abs(b).max(-1, keepdims=True) / 6.0)  # m 2^e, m in [1/2, 1)
    e = np.maximum(np.where(m == 0.5, e - 1, e), -126)
    e = np.where(np.abs(b).max(-1, keepdims=True) == 0, -126, e)
    v = np.abs(np.ldexp(b, -e))
    # nearest level, ties to the even code
    mid = (LEVELS[1:] + LEVELS[:-1]) / 2
    code = np.zeros(v.shape, np.uint8)
    for c, at in enumerate(mid):
        code += ((v >= at) if c % 2 else (v > at)).astype(np.uint8)
    code |= np.where(np.signbit(b), 8, 0).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)[..., 0]
    return np.where(bad, 0, code).astype(np.uint8).reshape(*x.shape[:-1], -1), scale


def packed(x):
    """The bytes as stored."""
    code, scale = encode(x)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8), scale


def decode(code, scale, cols):
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return (v.reshape(*v.shape[:-1], -1, 32) * s[..., None]).reshape(v.shape)[..., :cols]


def rounded(x):
    return decode(*encode(x), x.shape[-1])


def product_bound(a, b, extra=0.0):
    """How far a sum of K products in FP32, in any order, may be from a b^T: each
    of K additions is off by at most 2^-23 of the sum of magnitudes (a unit in
    the last place: the matrix instructions' own rounding is not documented),
    and the result by `extra` of itself."""
    return a.shape[-1] * 2.0**-23 * (np.abs(a) @ np.abs(b).T) + extra * np.abs(a @ b.T) + 1e-300


def route(x, k, bias=None, sigmoid=False, groups=1, kept=1, renorm=True, scale=1.0, lowest=-np.finfo(np.float32).max):
    """(ids, weights, gap): gap is the distance of the nearest two keys (or group
    keys) that decide anything, for judging which rows have a clear answer."""
    x = np.asarray(x, np.float64)
    tokens, experts = x.shape
    shut = ~(x > lowest)
    score, key = scores(x, sigmoid, lowest), np.where(shut, -np.inf, x)
    if bias is not None:
        key = np.where(shut, -np.inf, score + np.asarray(bias, np.float64))
    ids, weights, gap = np.full((tokens, k), -1, np.int32), np.zeros((tokens, k)), np.full(tokens, np.inf)

    def order(v):  # best first, ties to the lowest
        return sorted(range(len(v)), key=lambda i: (-v[i], i))

    def apart(v, o):
        d = [v[o[i]] - v[o[i + 1]] for i in range(len(o) - 1) if np.isfinite(v[o[i + 1]])]
        return min([d_ for d_ in d if d_ > 0], default=np.inf)

    for t in range(tokens):
        v = key[t].copy()
        if groups > 1:
            g = np.sort(v.reshape(groups, -1), 1)[:, ::-1]
            s = g[:, 0].copy()
            if bias is not None and g.shape[1] > 1:
                s = s + np.where(np.isfinite(g[:, 1]), g[:, 1], 0.0)
            o = order(s)
            gap[t] = min(gap[t], apart(s, o))
            v.reshape(groups, -1)[o[kept:]] = -np.inf
        o = order(v)
        gap[t] = min(gap[t], apart(v, o[: k + 1]))
        o = [e for e in o[:k] if v[e] > -np.inf]
        ids[t, : len(o)] = o
        w = score[t, o]
        weights[t, : len(o)] = (w / max(w.sum(), np.finfo(np.float32).tiny) if renorm else w) * scale
    return ids, weights, gap


def scores(x, sigmoid, lowest=-np.finfo(np.float32).max):
    x = np.asarray(x, np.float64)
    shut = ~(x > lowest)
    x = np.minimum(x, np.finfo(np.float32).max)
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            return np.where(shut, 0.0, 1.0 / (1.0 + np.exp(-x)))
        e = np.where(shut, 0.0, np.exp(x - np.where(shut, -np.inf, x).max(1, keepdims=True)))
    return e / np.maximum(e.sum(1, keepdims=True), 1.0)


def weights_of(x, ids, sigmoid, renorm, scale, lowest=-np.finfo(np.float32).max):
    """The weights of a fixed choice, a smooth function of the logits."""
    s = scores(x, sigmoid, lowest)
    w = np.where(ids >= 0, np.take_along_axis(s, np.maximum(ids, 0).astype(np.int64), 1), 0.0)
    return (w / np.maximum(w.sum(1, keepdims=True), np.finfo(np.float32).tiny) if renorm else w) * scale


def route_backward(x, ids, d_weights, sigmoid, renorm, scale, lowest=-np.finfo(np.float32).max):
    s = scores(x, sigmoid, lowest)
    at = np.maximum(ids, 0).astype(np.int64)
    real = ids >= 0
    w = np.where(real, np.take_along_axis(s, at, 1), 0.0)
    d = np.where(real, np.asarray(d_weights, np.float64) * scale, 0.0)
    if renorm:
        total = np.maximum(w.sum(1, keepdims=True), np.finfo(np.float32).tiny)
        d = np.where(real, (d - (d * w / total).sum(1, keepdims=True)) / total, 0.0)
    g = np.zeros_like(s)
    for j in range(ids.shape[1]):
        np.add.at(g, (np.arange(len(s)), at[:, j]), d[:, j])
    return g * s * (1.0 - s) if sigmoid else s * (g - (g * s).sum(1, keepdims=True))


def plan(ids, experts):
    flat = np.asarray(ids).reshape(-1)
    key = np.where((flat < 0) | (flat >= experts), experts, flat)
    order = np.argsort(key, kind="stable").astype(np.int32)
    offsets = np.searchsorted(key[order], np.arange(experts + 1)).astype(np.int32)
    return offsets, order


def experts_layer(x, ids, weights, w, d_out=None):
    """(y, out[, dx, d weights, dw]) of float64 x, w (experts x n x inputs, before
    rounding to MX4); weights are FP32."""
    tokens, k = ids.shape
    experts, n, inputs = w.shape
    xq = rounded(x)
    y = np.zeros((tokens, k, n))
    for t in range(tokens):
        for j in range(k):
            if 0 <= ids[t, j] < experts:
                y[t, j] = xq[t] @ rounded(w[ids[t, j]]).T
    real = (ids >= 0) & (ids < experts)
    wt = np.where(real, weights.astype(np.float64), 0.0)
    out = (y * wt[..., None]).sum(1)
    if d_out is None:
        return y, out
    dq = rounded(d_out)
    z = np.zeros((tokens, k, inputs))
    dw = np.zeros_like(w)
    for e in range(experts):
        t, j = np.nonzero(ids == e)
        if len(t) == 0:
            continue
        z[t, j] = dq[t] @ rounded(np.ascontiguousarray(w[e].T)).T
        g = (weights[t, j, None].astype(np.float32) * d_out[t].astype(np.float32)).astype(np.float64)
        dw[e] = rounded(np.ascontiguousarray(g.T)) @ rounded(np.ascontiguousarray(x[t].T)).T
    return y, out, (z * wt[..., None]).sum(1), (y * d_out[:, None]).sum(2), dw
