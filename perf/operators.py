"""Layers that compute in microscaled 4-bit floating point (MX4), as timed and compared cases.

Four groups of operators, through the public entry points of the library:

  encode   a matrix to MX4 along its rows, along its columns, or both in one
           pass (compressed activations and weights), and back to values;
  linear   the product of a dense layer whose operands are both MX4: a single
           token, a batch, a prompt, and a training step with the gradients of
           the input and of the weights;
  route    the choice of each token's experts from router logits, its weights
           and their gradient;
  experts  the layer of those experts: every token times the weights of each
           of its experts, joined by the routing weights, and its gradients.

MX4: blocks of 32 values share a power of two, the smallest at which no value
of the block lies above 6; a value is rounded to the nearest of 0, 0.5, 1, 1.5,
2, 3, 4, 6 (ties to the even code) and its sign.  A row's codes are padded with
zeros to a multiple of 256 values, two a byte, the first in the low half; the
scales are exponents biased by 127, one byte a block.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitsqueeze-llm_amd"))

own = False

_TYPES = {"f32": (0, torch.float32, 4), "bf16": (1, torch.bfloat16, 2), "f16": (2, torch.float16, 2)}


def _encode(name, rows, cols, type, both=False, ld=0):
    """ld: elements from one row to the next (0: cols)."""
    return {"name": name, "kind": "encode", "rows": rows, "cols": cols, "type": type, "both": both, "ld": ld or cols}


def _linear(name, tokens, inputs, outputs, type="bf16", out="bf16", train=False):
    return {"name": name, "kind": "linear", "tokens": tokens, "inputs": inputs, "outputs": outputs, "type": type,
            "out": out, "train": train}


def _route(name, tokens, experts, chosen, type="f32", scoring="softmax", bias=False, groups=1, kept=1, renorm=True,
           scale=1.0, masked=0.0, train=False):
    """masked: the share of tokens that may not use some of the experts."""
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "chosen": chosen, "type": type,
            "scoring": scoring, "bias": bias, "groups": groups, "kept": kept, "renorm": renorm, "scale": scale,
            "masked": masked, "train": train}


def _experts(name, tokens, experts, chosen, inputs, outputs, type="bf16", out="bf16", skew=1.0, train=False):
    """skew: how unevenly the experts are liked (0: evenly)."""
    return {"name": name, "kind": "experts", "tokens": tokens, "experts": experts, "chosen": chosen, "inputs": inputs,
            "outputs": outputs, "type": type, "out": out, "skew": skew, "train": train}


def listed():
    return [
        # a decode step's activations of a small batch: launches and host calls
        _encode("encode_small", 16, 4096, "bf16"),
        # a prompt's MLP activations kept for the backward pass, both directions
        _encode("encode_both", 4096, 11008, "bf16", both=True),
        # rows of an odd length, a slice of a wider FP32 matrix
        _encode("encode_ragged", 1000, 5003, "f32", both=True, ld=5008),
        # one token through an MLP's first product: the weights are read once
        _linear("linear_token", 1, 4096, 11008),
        # a decode batch of odd size through its second product
        _linear("linear_batch", 37, 11008, 4096),
        # a prompt
        _linear("linear_prefill", 4096, 4096, 11008),
        # a training step: weights encoded, forward, both gradients
        _linear("linear_train", 2048, 4096, 4096, train=True),
        # a decode step's routing
        _route("route_token", 16, 64, 4),
        # a training batch's routing: sigmoid scores, a bias for balance, groups
        _route("route_train", 16384, 256, 8, type="bf16", scoring="sigmoid", bias=True, groups=8, kept=4, scale=2.5,
               masked=0.02, train=True),
        # a decode batch through 32 experts: few rows each, some experts unused
        _experts("experts_token", 16, 32, 4, 4096, 2752),
        # a prompt through the same experts, some liked more than others
        _experts("experts_prefill", 4096, 32, 4, 4096, 2752),
        # a training step of a smaller layer
        _experts("experts_train", 2048, 16, 2, 2048, 2752, train=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: whole tiles, a multiple of eight, or any."""
    n = _log_uniform(rng, lo, hi)
    step = rng.choice((64, 8, 1))
    return int(min(hi, max(lo, round(n / step) * step)))


def draw(rng):
    # a bias only on logits of 16 bits: FP32 ones plus a bias come so near to each
    # other that the choice hangs on the last bit of exp
    kind = rng.choice(("encode", "linear", "linear", "route", "experts", "experts"))
    type = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "encode":
        cols = _size(rng, 64, 11008)
        c = _encode("", _size(rng, 1, 4096), cols, type, both=rng.random() < 0.5, ld=cols + rng.choice((0, 0, 5, 64)))
    elif kind == "linear":
        train = rng.random() < 0.3
        c = _linear("", _size(rng, 64, 2048) if train else _size(rng, 1, 4096), _size(rng, 64, 4096 if train else 11008),
                    _size(rng, 64, 4096), type=type, out=rng.choice(("bf16", "f32")), train=train)
    elif kind == "route":
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * rng.randint(2, 256 // groups)
        kept = rng.randint(1, groups)
        sigmoid = rng.random() < 0.5
        c = _route("", _size(rng, 1, 16384), experts, rng.randint(1, min(8, experts // groups * kept)), type=type,
                   scoring="sigmoid" if sigmoid else "softmax", bias=sigmoid and type != "f32", groups=groups, kept=kept,
                   renorm=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)), masked=rng.choice((0.0, 0.05)),
                   train=rng.random() < 0.5)
    else:
        train = rng.random() < 0.3
        experts = rng.randint(4, 16 if train else 32)
        c = _experts("", _size(rng, 32, 1024) if train else _size(rng, 1, 4096), experts, rng.randint(1, 4),
                     _size(rng, 64, 2048 if train else 4096), _size(rng, 64, 2752), type=type,
                     out=rng.choice(("bf16", "f32")), skew=rng.choice((0.0, 1.0, 2.0)), train=train)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs: what a program has in hand
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, cols, type, ld=0):
    """Normal values, one channel in 500 thirty times larger; rows ld apart."""
    ld = ld or cols
    x = _normal(g, rows, ld)
    x[:, torch.randperm(ld, device="cuda", generator=g)[: ld // 500]] *= 30.0
    return x.to(_TYPES[type][1])[:, :cols]


def _gradient(g, rows, cols, type):
    """Small, and smaller for some rows than for others."""
    return (_normal(g, rows, cols) * 0.02 * torch.exp(_normal(g, rows, 1))).to(_TYPES[type][1])


def _scale_bits(top):
    """The biased exponent of the smallest power of two that is at least top / 6
    (top: FP32, finite), at least 1."""
    return (((top.view(torch.int32) + 0x3FFFFF) >> 23) - 2).clamp_min(1)


def _power(bits):
    return (bits.to(torch.int32) << 23).view(torch.float32)


def _split(x):
    """Signed levels and the scales' exponents of FP32 x (... x cols), in blocks
    of 32 along the last axis, padded to a multiple of 256."""
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -cols % 256)).unflatten(-1, (-1, 32))
    bits = _scale_bits(x.abs().amax(-1, keepdim=True))
    v = x * _power(254 - bits)
    a = v.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, v), bits


def _rounded(x):
    """FP32 x to MX4 along its last axis and back."""
    v, bits = _split(x)
    return (v * _power(bits)).flatten(-2)[..., : x.shape[-1]]


def _pack(x):
    """The codes and scales of FP32 x, as bytes."""
    v, bits = _split(x)
    a = v.abs()
    code = torch.where(a < 2.0, a * 2.0, torch.where(a < 4.0, a + 2.0, a * 0.5 + 4.0)).to(torch.uint8)
    code = code + 8 * torch.signbit(v).to(torch.uint8)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] + 16 * code[..., 1]).contiguous(), bits.squeeze(-1).to(torch.uint8).contiguous()


def _unpack(packed, cols):
    """The FP32 values of codes and scales."""
    codes, scales = packed
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int32)
    levels = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0),
                          device=codes.device)
    v = levels[code].unflatten(-1, (-1, 32)) * _power(scales)[..., None]
    return v.flatten(-2)[..., :cols]


def _choices(g, tokens, experts, chosen, skew):
    """Different experts for each token, the liked ones more often; one token in
    fifty has none (padding).  int32 ids, FP32 weights that sum to one."""
    liked = -skew * torch.log(torch.arange(1, experts + 1, device="cuda").float())
    liked = liked[torch.randperm(experts, device="cuda", generator=g)]
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, device="cuda", generator=g).clamp(1e-9, 1 - 1e-7)))
    score, ids = torch.sort(liked + noise, dim=1, descending=True, stable=True)
    ids = ids[:, :chosen].to(torch.int32)
    weights = torch.softmax(score[:, :chosen], 1)
    none = torch.rand(tokens, 1, device="cuda", generator=g) < 0.02
    return torch.where(none, -1, ids).contiguous(), torch.where(none, 0.0, weights).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    s = {"case": case}
    if case["kind"] == "encode":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(g, rows, cols, case["type"], case["ld"])
        return s
    if case["kind"] == "route":
        tokens, experts, dtype = case["tokens"], case["experts"], _TYPES[case["type"]][1]
        logits = (_normal(g, tokens, experts) * 1.5 + 0.5 * _normal(g, 1, experts)).to(dtype)
        if case["masked"]:
            some = torch.rand(tokens, 1, device="cuda", generator=g) < case["masked"]
            closed = torch.rand(tokens, experts, device="cuda", generator=g) < 0.75
            logits = torch.where(some & closed, -math.inf, logits)
        s["logits"] = logits
        # moved a fixed step at a time by the balance rule
        s["bias"] = torch.round(_normal(g, experts) * 30.0) * 0.001 if case["bias"] else None
        s["d_weights"] = _normal(g, tokens, case["chosen"])
        return s
    inputs, outputs, tokens = case["inputs"], case["outputs"], case["tokens"]
    s["x"] = _activations(g, tokens, inputs, case["type"])
    if case["kind"] == "linear":
        w = _normal(g, outputs, inputs) * 0.02
    else:
        w = _normal(g, case["experts"], outputs, inputs) * 0.02
        s["ids"], s["weights"] = _choices(g, tokens, case["experts"], case["chosen"], case["skew"])
    if case["train"]:
        s["w"] = w.to(_TYPES[case["type"]][1])
        s["d_out"] = _gradient(g, tokens, outputs, case["type"])
    else:
        s["packed"] = _pack(w)  # laid out once, as a serving program keeps them
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _plain_encode(case, s):
    x, dtype = s["x"].float(), _TYPES[case["type"]][1]
    out = {"rows": _rounded(x).to(dtype)}
    if case["both"]:
        out["columns"] = _rounded(x.T.contiguous()).to(dtype)
    return out


def _plain_linear(case, s):
    dtype, x = _TYPES[case["out"]][1], s["x"].float()
    if not case["train"]:
        return (_rounded(x) @ _unpack(s["packed"], case["inputs"]).T).to(dtype)
    w, dy = s["w"].float(), s["d_out"].float()
    out = _rounded(x) @ _rounded(w).T
    dx = _rounded(dy) @ _rounded(w.T.contiguous()).T
    dw = _rounded(dy.T.contiguous()) @ _rounded(x.T.contiguous()).T
    return {"out": out.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}


def _plain_route(case, s):
    logits, bias, k = s["logits"], s["bias"], case["chosen"]
    x = logits.float()
    shut = (x <= torch.finfo(logits.dtype).min) | x.isnan()
    x = torch.where(shut, -math.inf, x).clamp_max(torch.finfo(torch.float32).max)
    if case["scoring"] == "sigmoid":
        score, rest = 1.0 / (1.0 + torch.exp(-x)), 1.0 / (1.0 + torch.exp(x))
    else:
        e = torch.where(shut, 0.0, torch.exp(x - x.amax(1, keepdim=True)))
        score = e / e.sum(1, keepdim=True).clamp_min(1.0)  # the largest is 1, or there is none
    score = torch.where(shut, 0.0, score)
    key = x if bias is None else torch.where(shut, -math.inf, score + bias)
    if case["groups"] > 1:
        grouped = key.unflatten(1, (case["groups"], -1))
        two = torch.sort(grouped, dim=2, descending=True).values[..., :2]
        of_group = two[..., 0]
        if bias is not None:
            of_group = of_group + torch.where(two[..., 1] == -math.inf, 0.0, two[..., 1])
        best = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, : case["kept"]]
        keep = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, best, True)
        key = torch.where(keep[..., None], grouped, -math.inf).flatten(1)
    key, ids = torch.sort(key, dim=1, descending=True, stable=True)
    ids, none = ids[:, :k], key[:, :k] == -math.inf
    chosen = torch.where(none, 0.0, score.gather(1, ids))
    total = chosen.sum(1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny) if case["renorm"] else 1.0
    out = {"ids": torch.where(none, -1, ids).to(torch.int32), "weights": chosen / total * case["scale"]}
    if case["train"]:
        d = torch.where(none, 0.0, s["d_weights"] * case["scale"])
        if case["renorm"]:
            d = (d - (d * (chosen / total)).sum(1, keepdim=True)) / total
        d = torch.where(none, 0.0, d)
        d = torch.zeros_like(score).scatter_add_(1, ids, d)
        if case["scoring"] == "sigmoid":
            d = d * score * rest
        else:
            d = score * (d - (d * score).sum(1, keepdim=True))
        out["d_logits"] = torch.where(shut, 0.0, d).to(logits.dtype)
    return out


def _plan(ids, experts):
    """Pairs (token, place) in the experts' order, those of no expert last; where
    each expert begins; each expert's pairs side by side, and which of them are."""
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=experts + 1)
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    most = max(32, int(-(-counts[:experts].max() // 32) * 32))
    place = torch.arange(most, device=ids.device)
    real = place < counts[:experts, None]
    pairs = order[(offsets[:experts, None] + place).clamp_max(flat.numel() - 1)]
    return order, offsets[: experts + 1], pairs, real


def _plain_experts(case, s):
    dtype, experts, k = _TYPES[case["out"]][1], case["experts"], case["chosen"]
    inputs, tokens = case["inputs"], case["tokens"]
    order, offsets, pairs, real = _plan(s["ids"], experts)
    token = pairs // k
    weights = torch.where(s["ids"] < 0, 0.0, s["weights"])
    w = s["w"].float() if case["train"] else _unpack(s["packed"], inputs)
    x = s["x"].float()

    def spread(v):  # rows of the pairs' tokens, zero where there is no pair
        return torch.where(real[..., None], v[token], 0.0)

    def gathered(v):  # back into the pairs' own order
        out = v.new_zeros(tokens * k, v.shape[-1])
        out[pairs[real]] = v[real]
        return out.unflatten(0, (tokens, k))

    def turned(v):
        return v.transpose(1, 2).contiguous()

    y = gathered(torch.bmm(spread(_rounded(x)), turned(_rounded(w) if case["train"] else w)))
    out = {"out": (y * weights[..., None]).sum(1).to(dtype), "offsets": offsets.to(torch.int32),
           "order": order.to(torch.int32)}
    if case["train"]:
        dy = s["d_out"].float()
        z = gathered(torch.bmm(spread(_rounded(dy)), turned(_rounded(turned(w)))))
        out["dx"] = (z * weights[..., None]).sum(1).to(dtype)
        out["d_weights"] = (y * dy[:, None]).sum(2)
        pair_dy = spread(dy) * torch.where(real, weights.reshape(-1)[pairs], 0.0)[..., None]
        out["dw"] = torch.bmm(_rounded(turned(pair_dy)), turned(_rounded(turned(spread(x))))).to(dtype)
    return out


# ---------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------
def _buffer(s, name, *shape, dtype=torch.uint8):
    """Outputs and workspaces, which a program keeps from step to step."""
    if name not in s:
        s[name] = torch.empty(shape, dtype=dtype, device="cuda")
    return s[name]


def _mx4_buffers(s, B, name, rows, cols, batch=1):
    return (_buffer(s, name + "_codes", batch * B.lib().bsq_mx4_codes_bytes(rows, cols)),
            _buffer(s, name + "_scales", batch * B.lib().bsq_mx4_scales_bytes(rows, cols)))


def _own_encode(case, s, B):
    L, stream, x = B.lib(), torch.cuda.current_stream().cuda_stream, s["x"]
    rows, cols, (t, dtype, _) = case["rows"], case["cols"], _TYPES[case["type"]]
    codes, scales = _mx4_buffers(s, B, "r", rows, cols)
    ct, st = _mx4_buffers(s, B, "c", cols, rows) if case["both"] else (None, None)
    B.check(L.bsq_mx4_encode(x.data_ptr(), t, 1, rows, cols, case["ld"], 0, codes.data_ptr(), scales.data_ptr(),
                             ct.data_ptr() if case["both"] else None, st.data_ptr() if case["both"] else None, stream),
            "mx4 encode")
    out = {"rows": _buffer(s, "rows", rows, cols, dtype=dtype)}
    B.check(L.bsq_mx4_decode(codes.data_ptr(), scales.data_ptr(), rows, cols, out["rows"].data_ptr(), t, cols, stream),
            "mx4 decode")
    if case["both"]:
        out["columns"] = _buffer(s, "columns", cols, rows, dtype=dtype)
        B.check(L.bsq_mx4_decode(ct.data_ptr(), st.data_ptr(), cols, rows, out["columns"].data_ptr(), t, rows, stream),
                "mx4 decode")
    return out


def _own_linear(case, s, B):
    L, stream, x = B.lib(), torch.cuda.current_stream().cuda_stream, s["x"]
    m, k, n = case["tokens"], case["inputs"], case["outputs"]
    t, (o, dtype, _) = _TYPES[case["type"]][0], _TYPES[case["out"]]
    if "work" not in s:
        size = L.bsq_mx4_linear_backward_workspace(m, n, k) if case["train"] else 0
        _buffer(s, "work", max(size, L.bsq_mx4_linear_workspace(m, n, k)))
    work, out = s["work"], _buffer(s, "out", m, n, dtype=dtype)
    xt = xs = None
    if case["train"]:
        codes, scales = _mx4_buffers(s, B, "wr", n, k)
        ct, st = _mx4_buffers(s, B, "wc", k, n)
        B.check(L.bsq_mx4_encode(s["w"].data_ptr(), t, 1, n, k, k, 0, codes.data_ptr(), scales.data_ptr(),
                                 ct.data_ptr(), st.data_ptr(), stream), "mx4 encode")
        xt, xs = (b.data_ptr() for b in _mx4_buffers(s, B, "xc", k, m))
    else:
        codes, scales = s["packed"]
    B.check(L.bsq_mx4_linear(x.data_ptr(), t, m, k, k, codes.data_ptr(), scales.data_ptr(), n, out.data_ptr(), o, n, xt,
                             xs, work.data_ptr(), work.numel(), stream), "mx4 linear")
    if not case["train"]:
        return out
    dx, dw = _buffer(s, "dx", m, k, dtype=dtype), _buffer(s, "dw", n, k, dtype=dtype)
    B.check(L.bsq_mx4_linear_backward(s["d_out"].data_ptr(), t, m, n, n, xt, xs, ct.data_ptr(), st.data_ptr(), k,
                                      dx.data_ptr(), k, dw.data_ptr(), k, o, work.data_ptr(), work.numel(), stream),
            "mx4 linear backward")
    return {"out": out, "dx": dx, "dw": dw}


def _own_route(case, s, B):
    L, stream, logits = B.lib(), torch.cuda.current_stream().cuda_stream, s["logits"]
    tokens, experts, k, t = case["tokens"], case["experts"], case["chosen"], _TYPES[case["type"]][0]
    ids, weights = _buffer(s, "ids", tokens, k, dtype=torch.int32), _buffer(s, "weights", tokens, k, dtype=torch.float32)
    scoring = 1 if case["scoring"] == "sigmoid" else 0
    B.check(L.bsq_moe_route(logits.data_ptr(), t, tokens, experts, experts,
                            s["bias"].data_ptr() if case["bias"] else None, scoring, case["groups"], case["kept"], k,
                            case["renorm"], case["scale"], ids.data_ptr(), weights.data_ptr(), stream), "moe route")
    out = {"ids": ids, "weights": weights}
    if case["train"]:
        out["d_logits"] = _buffer(s, "d_logits", tokens, experts, dtype=logits.dtype)
        B.check(L.bsq_moe_route_backward(logits.data_ptr(), t, tokens, experts, experts, scoring, k, case["renorm"],
                                         case["scale"], ids.data_ptr(), s["d_weights"].data_ptr(),
                                         out["d_logits"].data_ptr(), experts, stream), "moe route backward")
    return out


def _own_experts(case, s, B):
    L, stream, x = B.lib(), torch.cuda.current_stream().cuda_stream, s["x"]
    m, k, n, e, c = case["tokens"], case["inputs"], case["outputs"], case["experts"], case["chosen"]
    t, (o, dtype, _) = _TYPES[case["type"]][0], _TYPES[case["out"]]
    y_type = 0 if case["train"] else o  # the gradient of the weights is an FP32 sum over y
    if "work" not in s:
        size = L.bsq_moe_linear_backward_workspace(m, c, n, k, e) if case["train"] else 0
        _buffer(s, "work", max(size, L.bsq_moe_linear_workspace(m, c, n, k, e)))
    work, out = s["work"], _buffer(s, "out", m, n, dtype=dtype)
    y = _buffer(s, "y", m * c, n, dtype=torch.float32 if case["train"] else dtype)
    offsets, order = _buffer(s, "offsets", e + 1, dtype=torch.int32), _buffer(s, "order", m * c, dtype=torch.int32)
    if case["train"]:
        codes, scales = _mx4_buffers(s, B, "wr", n, k, e)
        ct, st = _mx4_buffers(s, B, "wc", k, n, e)
        B.check(L.bsq_mx4_encode(s["w"].data_ptr(), t, e, n, k, k, n * k, codes.data_ptr(), scales.data_ptr(),
                                 ct.data_ptr(), st.data_ptr(), stream), "mx4 encode")
    else:
        codes, scales = s["packed"]
    B.check(L.bsq_moe_linear(x.data_ptr(), t, m, k, k, s["ids"].data_ptr(), s["weights"].data_ptr(), c,
                             codes.data_ptr(), scales.data_ptr(), e, n, offsets.data_ptr(), order.data_ptr(),
                             y.data_ptr(), y_type, out.data_ptr(), o, n, work.data_ptr(), work.numel(), stream),
            "moe linear")
    got = {"out": out, "offsets": offsets, "order": order}
    if case["train"]:
        got["dx"], got["dw"] = _buffer(s, "dx", m, k, dtype=dtype), _buffer(s, "dw", e, n, k, dtype=dtype)
        got["d_weights"] = _buffer(s, "d_weights", m, c, dtype=torch.float32)
        B.check(L.bsq_moe_linear_backward(s["d_out"].data_ptr(), t, m, n, n, x.data_ptr(), t, k, k, s["ids"].data_ptr(),
                                          s["weights"].data_ptr(), c, offsets.data_ptr(), order.data_ptr(),
                                          y.data_ptr(), y_type, ct.data_ptr(), st.data_ptr(), e, got["dx"].data_ptr(),
                                          k, got["d_weights"].data_ptr(), got["dw"].data_ptr(), o, work.data_ptr(),
                                          work.numel(), stream), "moe linear backward")
    return got


def run(state):
    kind = state["case"]["kind"]
    if own:
        import bitsqz_amd as B

        form = {"encode": _own_encode, "linear": _own_linear, "route": _own_route, "experts": _own_experts}[kind]
        return form(state["case"], state, B)
    form = {"encode": _plain_encode, "linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}[kind]
    return form(state["case"], state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _packed_bytes(rows, cols):
    return rows * -(-cols // 256) * 136


def work(case):
    size = _TYPES[case["type"]][2]
    if case["kind"] == "encode":
        rows, cols = case["rows"], case["cols"]
        packed = _packed_bytes(rows, cols) + (_packed_bytes(cols, rows) if case["both"] else 0)
        return {"bytes": rows * cols * size * (3 if case["both"] else 2) + 2 * packed, "flops": 0}
    if case["kind"] == "route":
        tokens, experts, k = case["tokens"], case["experts"], case["chosen"]
        b = tokens * experts * size + tokens * k * 8
        if case["train"]:
            b += tokens * experts * size + tokens * k * 4
        return {"bytes": b, "flops": 0}
    m, k, n, o = case["tokens"], case["inputs"], case["outputs"], _TYPES[case["out"]][2]
    pairs = m * case.get("chosen", 1)
    matrices = 1.0
    if case["kind"] == "experts":  # the experts that an even choice uses
        matrices = case["experts"] * (1.0 - (1.0 - case["chosen"] / case["experts"]) ** m if case["chosen"] < case["experts"] else 1.0)
    flops = 2.0 * pairs * k * n
    b = m * k * size + m * n * o + pairs * (8 if case["kind"] == "experts" else 0)
    if not case["train"]:
        return {"bytes": b + matrices * _packed_bytes(n, k), "flops": flops}
    every = case.get("experts", 1)
    return {"bytes": b + every * n * k * (size + o) + m * n * size + m * k * o, "flops": 3.0 * flops}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _two_to(exponent):
    """FP64 powers of two, from their bits."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _mx4(x):
    """FP64 x through MX4 along its last axis."""
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -cols % 32)).reshape(*x.shape[:-1], -1, 32)
    top = x.abs().amax(-1, keepdim=True) / 6.0
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [1/2, 1)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp_min(-126)
    v = x * _two_to(-exponent)
    a = v.abs()
    level = torch.zeros_like(a)
    # from one level to the next: at the midpoint, which goes to the even code
    for mid, gap, up in ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False), (1.75, 0.5, True), (2.5, 1.0, False),
                         (3.5, 1.0, True), (5.0, 2.0, False)):
        level += gap * ((a >= mid) if up else (a > mid))
    return (level * v.sign() * _two_to(exponent)).reshape(*x.shape[:-2], -1)[..., :cols]


def _unpacked(packed, cols):
    codes, scales = packed
    levels = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), dtype=torch.float64, device=codes.device)
    nibbles = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.uint8, device=codes.device)
    nibbles[..., 0::2] = codes % 16
    nibbles[..., 1::2] = codes // 16
    v = levels[(nibbles % 8).long()] * (1.0 - 2.0 * (nibbles >= 8))
    return (v * _two_to(scales.to(torch.int64) - 127).repeat_interleave(32, -1))[..., :cols]


def _exact_experts(case, s):
    tokens, k, experts = case["tokens"], case["chosen"], case["experts"]
    x = s["x"].double()
    ids, weights = s["ids"].long(), s["weights"].double()
    out = x.new_zeros(tokens, case["outputs"])
    train = case["train"]
    xq = _mx4(x)
    if train:
        dy = s["d_out"].double()
        dyq = _mx4(dy)
        dx, dw = torch.zeros_like(x), x.new_zeros(experts, case["outputs"], case["inputs"])
        d_weights = torch.zeros_like(weights)
    for e in range(experts):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        w = s["w"][e].double() if train else _unpacked((s["packed"][0][e], s["packed"][1][e]), case["inputs"])
        y = xq[t] @ (_mx4(w) if train else w).T
        out.index_add_(0, t, y * weights[t, j, None])
        if train:
            dx.index_add_(0, t, dyq[t] @ _mx4(w.T).T * weights[t, j, None])
            d_weights[t, j] = (y * dy[t]).sum(1)
            # the weighted gradient is held in FP32 before it is rounded to MX4
            dw[e] = _mx4((s["weights"][t, j, None] * s["d_out"][t].float()).double().T) @ _mx4(x[t].T).T
    got = {"out": out, "offsets": None, "order": None}
    if train:
        got |= {"dx": dx, "d_weights": d_weights, "dw": dw}
    return got


def _exact_route(case, s):
    x, k = s["logits"].double(), case["chosen"]
    shut = ~(x > torch.finfo(s["logits"].dtype).min)
    if case["scoring"] == "sigmoid":
        score = torch.sigmoid(x)
    else:
        score = torch.softmax(torch.where(shut, -1e300, x), 1)
    score = score.masked_fill(shut, 0.0)
    key = (score + (s["bias"].double() if case["bias"] else 0.0)) if case["bias"] else x
    key = key.masked_fill(shut, -math.inf)
    groups, each = case["groups"], case["experts"] // case["groups"]
    if groups > 1:
        by = key.reshape(-1, groups, each).topk(2 if case["bias"] else 1, dim=2).values
        by = torch.where(by[..., :1] == -math.inf, -math.inf, by.masked_fill(by == -math.inf, 0.0).sum(2, keepdim=True))
        last = by.squeeze(2).argsort(dim=1, descending=True, stable=True)[:, case["kept"]:]
        away = torch.zeros(key.shape[0], groups, dtype=torch.bool, device=key.device)
        away[torch.arange(key.shape[0], device=key.device)[:, None], last] = True
        key = key.masked_fill(away.repeat_interleave(each, 1), -math.inf)
    ids = key.argsort(dim=1, descending=True, stable=True)[:, :k]
    taken = torch.zeros_like(shut).scatter(1, ids, True) & (key > -math.inf)
    part = score * taken
    total = part.sum(1, keepdim=True) if case["renorm"] else torch.ones_like(part[:, :1])
    share = torch.where(total > 0, part / total, 0.0) * case["scale"]
    got = {"ids": None, "weights": share.gather(1, ids)}
    if case["train"]:
        d = torch.zeros_like(score).scatter(1, ids, s["d_weights"].double() * case["scale"]) * taken
        if case["renorm"]:
            d = torch.where(total > 0, (d - (d * part / total).sum(1, keepdim=True)) / total, 0.0) * taken
        if case["scoring"] == "sigmoid":
            got["d_logits"] = torch.where(shut, 0.0, d * score * torch.sigmoid(-x))
        else:
            got["d_logits"] = score * (d - (d * score).sum(1, keepdim=True))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "encode":
        x = s["x"].double()
        return {"rows": _mx4(x), "columns": _mx4(x.T)} if case["both"] else {"rows": _mx4(x)}
    if case["kind"] == "route":
        return _exact_route(case, s)
    if case["kind"] == "experts":
        return _exact_experts(case, s)
    x = s["x"].double()
    if not case["train"]:
        return _mx4(x) @ _unpacked(s["packed"], case["inputs"]).T
    w, dy = s["w"].double(), s["d_out"].double()
    return {"out": _mx4(x) @ _mx4(w).T, "dx": _mx4(dy) @ _mx4(w.T).T, "dw": _mx4(dy.T) @ _mx4(x.T).T}
