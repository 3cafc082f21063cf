"""Attention over a paged cache of keys and values in 4 bits, as timed and compared cases.

Four groups of operators, through the public entry points of the library:

  plan       the bookkeeping of a step, on the GPU: from the requests' lengths
             the pages that each takes from a stack of free ones, its table of
             pages, and every new token's request, position and slot;
  rope       rotary positions of queries and keys, the pairs' halves side by
             side or a half apart, part of the head, stretched for long
             contexts, and their gradient;
  append     a step's keys and values into the cache: queries and keys rotated,
             keys and values packed to 4 bits at their slots; and read back;
  attention  of single tokens, chunks and whole prompts over such a cache.

The cache holds microscaled 4-bit values (MX4): blocks of 32 values along a head
share a power of two, the smallest at which no value of the block lies above 6;
a value is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even
code) and its sign.  A page holds `page` tokens; for each head of keys and values
it has the keys' codes, the values' codes (a token's row: two codes a byte, the
first in the low half, padded with zeros to whole blocks), the keys' scales and
the values' scales, bytes biased by 127: 16 tokens side by side, that of token t
and block b at 4 (blocks (t % 4) + b) + t % 16 / 4.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitsqueeze-llm_amd"))

own = False

_TYPES = {"f32": (0, torch.float32, 4), "bf16": (1, torch.bfloat16, 2), "f16": (2, torch.float16, 2)}


def _plan(name, requests, page, past, new, prompts=0.0, ended=0.0, spare=0):
    """past: the longest context so far; new: a prompt's tokens, for the share
    `prompts` of the requests (the others have one); ended: the share that ends;
    spare: pages that stay free (below zero: those that are missing)."""
    return {"name": name, "kind": "plan", "requests": requests, "page": page, "past": past, "new": new,
            "prompts": prompts, "ended": ended, "spare": spare}


def _rope(name, tokens, heads, dim, dims, type="bf16", interleaved=False, base=10000.0, stretch=1.0, far=4096, pad=0,
          train=False):
    """dims: of the head's values, those that turn; stretch: of the context's
    length; far: the positions' range; pad: elements between two tokens' rows."""
    return {"name": name, "kind": "rope", "tokens": tokens, "heads": heads, "dim": dim, "dims": dims, "type": type,
            "interleaved": interleaved, "base": base, "stretch": stretch, "far": far, "pad": pad, "train": train}


def _append(name, tokens, queries, heads, dim, page, type="bf16", interleaved=False, base=10000.0, stretch=1.0, far=4096,
            absent=0):
    """queries, heads: of the queries, and of keys and values; absent: rows
    behind the last token."""
    return {"name": name, "kind": "append", "tokens": tokens, "queries": queries, "heads": heads, "dim": dim, "page": page,
            "type": type, "interleaved": interleaved, "base": base, "stretch": stretch, "far": far, "absent": absent}


def _attention(name, requests, lo, hi, queries, heads, dim, page=16, new=1, chunks=0, type="bf16", out="bf16", window=0):
    """lo, hi: cached tokens, spread over their logarithm; new: the tokens of
    `chunks` of the requests (the others have one)."""
    return {"name": name, "kind": "attention", "requests": requests, "lo": lo, "hi": hi, "queries": queries, "heads": heads,
            "dim": dim, "page": page, "new": new, "chunks": chunks, "type": type, "out": out, "window": window}


def listed():
    return [
        # a decode step's bookkeeping: one launch
        _plan("plan_decode", 64, 16, 8192, 1, ended=0.03, spare=500),
        # a busy server's step: decoding requests, new prompts, ended ones
        _plan("plan_mixed", 2000, 32, 16384, 1500, prompts=0.02, ended=0.02, spare=3000),
        # queries and keys of a decode step, side by side in one row
        _rope("rope_token", 16, 40, 128, 128),
        # a training batch's queries: half of the head turned, far positions, forward and gradient
        _rope("rope_train", 8192, 32, 128, 64, interleaved=True, base=500000.0, stretch=8.0, far=1 << 20, train=True),
        # a decode batch's queries, keys and values, some rows behind the last
        _append("append_token", 37, 32, 8, 128, 16, absent=27),
        # a prompt's, stretched positions, an odd number of tokens
        _append("append_prompt", 8191, 32, 8, 128, 64, base=500000.0, stretch=4.0, far=131072),
        # a decode step of a small batch over short contexts: launches count
        _attention("attention_token", 16, 400, 1200, 32, 8, 128),
        # few requests over very long contexts
        _attention("attention_long", 8, 40000, 90000, 32, 8, 128, page=64),
        # a server's decode batch: contexts of all lengths
        _attention("attention_ragged", 128, 16, 16384, 32, 8, 128),
        # a prompt
        _attention("attention_prompt", 1, 0, 0, 32, 8, 128, page=64, new=8192, chunks=1),
        # prompts in chunks beside decoding requests, in a window, FP16
        _attention("attention_chunks", 24, 500, 8000, 20, 4, 96, page=32, new=500, chunks=5, type="f16", out="f16",
                   window=4096),
        # a few tokens to verify for each request, one head of keys to a query's, FP32
        _attention("attention_verify", 9, 100, 5000, 12, 12, 64, new=5, chunks=9, type="f32", out="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: a multiple of 16, or any."""
    n = _log_uniform(rng, lo, hi)
    step = rng.choice((16, 1, 1))
    return int(min(hi, max(lo, round(n / step) * step)))


def draw(rng):
    kind = rng.choice(("plan", "rope", "append", "attention", "attention", "attention"))
    type = rng.choice(("bf16", "bf16", "f16", "f32"))
    page = rng.choice((16, 32, 64, 128, 256))
    dim = rng.choice((64, 64, 80, 96, 112, 128, 128, 128, 192, 256, 8 * rng.randint(4, 32)))
    stretch = dict(base=rng.choice((10000.0, 500000.0)), stretch=rng.choice((1.0, 1.0, 4.0, 16.0)),
                   far=int(_log_uniform(rng, 1000, 1 << 20)), interleaved=rng.random() < 0.4)
    if kind == "plan":
        c = _plan("", _size(rng, 1, 2000), page, _size(rng, 64, 16384), _size(rng, 1, 1500),
                  prompts=rng.choice((0.0, 0.02, 0.02)), ended=rng.choice((0.0, 0.03, 0.1)),
                  spare=rng.choice((500, 2000, 0, -3)))
    elif kind == "rope":
        tokens = _size(rng, 1, 8192)
        c = _rope("", tokens, min(64, rng.randint(1, 64), 8192 * 4096 // (tokens * dim) or 1), dim,
                  rng.choice((dim, dim, dim // 2 // 2 * 2, 32)), type=type, pad=rng.choice((0, 0, 3, 64)),
                  train=rng.random() < 0.5, **stretch)
    elif kind == "append":
        heads = rng.choice((1, 2, 4, 8))
        tokens = _size(rng, 1, 8191)
        c = _append("", tokens, heads * rng.randint(1, max(1, min(8, 8191 * 4096 // (tokens * heads * dim)))), heads, dim,
                    page, type=type, absent=rng.choice((0, 0, 5, 32)), **stretch)
    else:
        group = rng.choice((1, 2, 3, 4, 4, 5, 8, 16))
        heads = rng.choice((1, 2, 4, 8))
        short = rng.random() < 0.6
        requests = _size(rng, 1, 128)
        # what the padded plain form holds: keys, and scores
        most = int(min(65536, 1.0e9 / (requests * heads * dim)))
        new = 1 if short else _size(rng, 2, 2000)
        chunks = 0 if short else rng.randint(1, min(4, requests))
        if not short:
            most = max(64, int(min(most, 8192, 0.5e9 / (requests * new * heads * group))))
        hi = _size(rng, 16, max(17, most))
        c = _attention("", requests, rng.choice((0, 1, max(1, hi // 8), hi)), hi, heads * group, heads, dim, page=page,
                       new=new, chunks=chunks, type=type, out=rng.choice((type, type, "f32")),
                       window=rng.choice((0, 0, 0, _size(rng, 1, 4096))))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs: what a program has in hand
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly over the logarithm of one more."""
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * (i + 0.5) / n) - 1)) for i in range(n)]


def _lengths(case):
    """(cached, new) tokens of each request; new below zero: it has ended."""
    n = case["requests"]
    if case["kind"] == "plan":
        past = _spread(n, 1, case["past"])
        prompts, ended = int(round(n * case["prompts"])), int(round(n * case["ended"]))
        new = [case["new"] - 7 * i % 50 if case["new"] > 50 else case["new"] for i in range(prompts)] + [1] * (n - prompts)
        pairs = [(0, m) if i < prompts else (p, m) for i, (p, m) in enumerate(zip(past, new))]
        return [(p, -1) if i >= n - ended else (p, m) for i, (p, m) in enumerate(pairs)]
    past = _spread(n, case["lo"], case["hi"])
    step = n / max(1, case["chunks"])
    chunk = {int(i * step) for i in range(case["chunks"])}
    return [(p, case["new"] if i in chunk else 1) for i, p in enumerate(past)]


def _pages(tokens, page):
    return -(-tokens // page)


def _frequencies(dims, base, stretch):
    """The angles' steps from position to position, FP64, and the length of what
    is turned.  Stretched by parts: pairs that turn less than once over 4096
    positions are slowed by `stretch`, those that turn over 32 times are not, with
    a ramp between; lengths grow with the logarithm of `stretch`."""
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if stretch == 1.0:
        return f, 1.0

    def pair(turns):  # the pair that turns so often over 4096 positions
        return dims * math.log(4096 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = max(0.0, math.floor(pair(32.0))), min(dims - 1.0, math.ceil(pair(1.0)))
    keep = [1.0 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(dims // 2)]
    return [x * (k + (1.0 - k) / stretch) for x, k in zip(f, keep)], 0.1 * math.log(stretch) + 1.0


def _scale_bits(top):
    """The biased exponent of the smallest power of two that is at least top / 6
    (top: FP32, finite), at least 1."""
    return (((top.view(torch.int32) + 0x3FFFFF) >> 23) - 2).clamp_min(1)


def _power(bits):
    return (bits.to(torch.int32) << 23).view(torch.float32)


def _split(x):
    """Signed levels and the scales' exponents of FP32 x, in blocks of 32 along
    the last axis."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    bits = _scale_bits(x.abs().amax(-1, keepdim=True))
    v = x * _power(254 - bits)
    a = v.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, v), bits


def _rounded(x):
    """FP32 x to MX4 along its last axis and back."""
    v, bits = _split(x)
    return (v * _power(bits)).flatten(-2)[..., : x.shape[-1]]


def _packed(x):
    """FP32 x (pages x heads x tokens x dim) as the cache holds it: codes and
    scales, pages x heads x bytes."""
    v, bits = _split(x)
    a = v.abs()
    code = torch.where(a < 2.0, a * 2.0, torch.where(a < 4.0, a + 2.0, a * 0.5 + 4.0)).to(torch.uint8)
    code = (code + 8 * torch.signbit(v).to(torch.uint8)).flatten(-2).unflatten(-1, (-1, 2))
    scales = bits.squeeze(-1).to(torch.uint8).unflatten(2, (-1, 4, 4)).permute(0, 1, 2, 4, 5, 3)
    return (code[..., 0] + 16 * code[..., 1]).flatten(2), scales.flatten(2)


def _cache(g, pages, page, heads, dim):
    """A cache in use: keys of which some channels are larger, values."""
    k = _normal(g, pages, heads, page, dim)
    k *= torch.where(torch.rand(heads, 1, dim, device="cuda", generator=g) < 0.03, 4.0, 1.0)
    k, ks = _packed(k)
    v, vs = _packed(_normal(g, pages, heads, page, dim))
    return torch.cat((k, v, ks, vs), -1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 31)
    s = {"case": case}

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def drawn(n, of):
        return torch.randperm(of, device="cuda", generator=g)[:n].to(torch.int32)

    if case["kind"] in ("plan", "attention"):
        pairs, page = _lengths(case), case["page"]
        random.Random(int(seed)).shuffle(pairs)
        now = [p + max(m, 0) for p, m in pairs]
        width = max(1, _pages(max(now), page)) + 3
        if case["kind"] == "plan":
            held = [_pages(p, page) for p, _ in pairs]
            need = sum(_pages(n, page) - h for n, h, (_, m) in zip(now, held, pairs) if m >= 0)
            freed = sum(h for h, (_, m) in zip(held, pairs) if m < 0)
            free = max(0, need - freed + case["spare"])
            pages = sum(held) + free
            total = sum(max(m, 0) for _, m in pairs)
            s["tokens"] = -(-total // 64) * 64  # of the captured step
        else:
            held, pages = [_pages(n, page) for n in now], sum(_pages(n, page) for n in now) + 5
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((len(pairs), width), -1, dtype=torch.int32, device="cuda")
        place = torch.arange(width, device="cuda")
        table[place < ints(held)[:, None]] = order[: sum(held)]
        s["table"], s["pages"] = table, pages
        s["new"] = ints([m for _, m in pairs])
        if case["kind"] == "plan":
            s["lengths"] = ints([p for p, _ in pairs])
            s["free"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
            s["free"][:free] = order[sum(held):]
            s["count"] = ints([free])
            return s
        s["lengths"] = ints(now)
        s["starts"] = torch.nn.functional.pad(s["new"].cumsum(0), (1, 0)).to(torch.int32)
        s["cache"] = _cache(g, pages, page, case["heads"], case["dim"])
        q = _normal(g, sum(m for _, m in pairs), case["queries"], case["dim"]) * 1.5
        s["q"] = q.to(_TYPES[case["type"]][1])
        s["scale"] = case["dim"] ** -0.5
        return s
    dtype, tokens, dim = _TYPES[case["type"]][1], case["tokens"], case["dim"]
    dims = case.get("dims", dim)
    f, s["factor"] = _frequencies(dims, case["base"], case["stretch"])
    s["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    s["positions"] = torch.randint(case["far"], (tokens,), device="cuda", generator=g).to(torch.int32)
    if case["kind"] == "rope":
        width = case["heads"] * dim
        s["x"] = _normal(g, tokens, width + case["pad"]).to(dtype)[:, :width]
        s["d_out"] = (_normal(g, tokens, width) * 0.02).to(dtype)
        return s
    # one product's rows: queries, keys, values
    rows = tokens + case["absent"]
    width = (case["queries"] + 2 * case["heads"]) * dim
    x = _normal(g, rows, width)
    keys = slice(case["queries"] * dim, (case["queries"] + case["heads"]) * dim)
    x[:, keys] *= torch.where(torch.rand(keys.stop - keys.start, device="cuda", generator=g) < 0.03, 4.0, 1.0)
    s["x"] = x.to(dtype)
    s["pages"] = _pages(tokens, case["page"]) + 9
    taken = drawn(_pages(tokens, case["page"]), s["pages"])
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    s["slots"] = taken[(at // case["page"]).long()] * case["page"] + at % case["page"]
    gone = ints([-1] * case["absent"])
    s["slots"], s["positions"] = torch.cat((s["slots"], gone)), torch.cat((s["positions"], gone))
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _plain_plan(case, s):
    page, table, free = case["page"], s["table"].long(), s["free"].long()
    requests, width = table.shape
    pages, tokens = s["pages"], s["tokens"]
    past, new, place = s["lengths"].long(), s["new"].long(), torch.arange(width, device="cuda")
    held = (past + page - 1) // page
    # pages of the ended ones onto the stack
    freed = (new < 0)[:, None] & (place < held[:, None])
    top = s["count"][0].long() + freed.sum()
    to = s["count"].long() + freed.flatten().cumsum(0).view_as(freed) - 1
    stack = torch.nn.functional.pad(free, (0, 1))
    stack[torch.where(freed, to, pages)] = table
    # pages for the new tokens, request by request from its top
    n = new.clamp_min(0)
    need = torch.where(new < 0, 0, (past + n + page - 1) // page - held)
    last = need.cumsum(0)
    served = (new >= 0) & ((need == 0) | (last <= top))
    first = last - need
    starts = torch.nn.functional.pad(n.cumsum(0), (1, 0))
    taken = served[:, None] & (place >= held[:, None]) & (place < (held + need)[:, None])
    table = torch.where(taken, stack[(top - 1 - (first - held)[:, None] - place).clamp(0, pages)], table)
    # the tokens
    t = torch.arange(tokens, device="cuda")
    r = torch.searchsorted(starts[1:], t, right=True)
    real = r < requests
    r = r.clamp_max(requests - 1)
    placed = real & served[r]
    position = past[r] + t - starts[r]
    slot = table[r, (position // page).clamp_max(width - 1)] * page + position % page
    left = torch.stack((top - torch.where(served, need, 0).sum(), (~served & (new >= 0)).sum()))
    out = {"starts": starts, "lengths": torch.where(new < 0, 0, torch.where(served, past + n, past)), "table": table,
           "left": left, "requests": torch.where(real, r, -1),
           "positions": torch.where(placed, position, -1), "slots": torch.where(placed, slot, -1)}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _turned(x, positions, s, dims, interleaved, back=False):
    """x (tokens x heads x dim), its first `dims` values turned, in FP64."""
    angle = positions.double()[:, None, None] * s["frequencies"]
    cos, sin = torch.cos(angle) * s["factor"], torch.sin(angle) * (-s["factor"] if back else s["factor"])
    x = x.double()
    if interleaved:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
    else:
        a, b = x[..., : dims // 2], x[..., dims // 2: dims]
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, x[..., dims:]), -1)


def _plain_rope(case, s):
    dtype, shape = _TYPES[case["type"]][1], (case["tokens"], case["heads"], case["dim"])
    out = {"out": _turned(s["x"].reshape(shape), s["positions"], s, case["dims"], case["interleaved"])}
    if case["train"]:
        out["dx"] = _turned(s["d_out"].reshape(shape), s["positions"], s, case["dims"], case["interleaved"], back=True)
    return {k: v.flatten(1).to(dtype) for k, v in out.items()}


def _parts(case, x):
    """Queries, keys and values of the product's rows."""
    x = x[: case["tokens"]].unflatten(1, (-1, case["dim"]))
    return x[:, : case["queries"]], x[:, case["queries"]: -case["heads"]], x[:, -case["heads"]:]


def _plain_append(case, s):
    dtype, dim = _TYPES[case["type"]][1], case["dim"]
    q, k, v = _parts(case, s["x"])
    positions = s["positions"][: case["tokens"]]
    # turned keys are held in their own type before they are packed
    q, k = (_turned(x, positions, s, dim, case["interleaved"]).to(dtype) for x in (q, k))
    return {"q": q.flatten(1), "k": _rounded(k.float()).flatten(1).to(dtype), "v": _rounded(v.float()).flatten(1).to(dtype)}


def _unpacked(codes, scales, page, dim):
    """FP32 values (... x tokens x dim) of the codes and scales of pages."""
    blocks = -(-dim // 32)
    codes = codes.unflatten(-1, (page, 16 * blocks))
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int32)
    levels = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0),
                          device=codes.device)
    scale = _power(scales.unflatten(-1, (page // 16, 4, blocks, 4)).movedim(-1, -3).flatten(-4, -2))
    return (levels[code].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)[..., :dim]


def _gathered(case, s):
    """Keys and values of each request in order, requests x heads x tokens x dim."""
    page, dim, blocks = case["page"], case["dim"], -(-case["dim"] // 32)
    most = _pages(max(p + m for p, m in _lengths(case)), page)
    held = s["cache"][s["table"][:, :most].clamp_min(0).long()].transpose(1, 2)  # requests x heads x pages x bytes
    row, scale = 16 * blocks * page, blocks * page
    k, v, ks, vs = held.split((row, row, scale, scale), -1)
    return _unpacked(k, ks, page, dim).flatten(2, 3), _unpacked(v, vs, page, dim).flatten(2, 3)


def _plain_attention(case, s):
    dtype, heads, group = _TYPES[case["out"]][1], case["heads"], case["queries"] // case["heads"]
    k, v = _gathered(case, s)
    requests, _, keys, dim = k.shape
    most = max(m for _, m in _lengths(case))
    # queries, padded to the longest chunk: requests x heads x (tokens, group) x dim
    i = torch.arange(most, device="cuda")
    t = (s["starts"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1).long()
    q = s["q"].float()[t].unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    del k
    at = (s["lengths"] - s["new"])[:, None] + i  # the queries' positions
    j = torch.arange(keys, device="cuda")
    seen = (j <= at[..., None]) & (j < s["lengths"][:, None, None])
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(-1, -1, -1, group, -1).flatten(2, 3)
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, v) / torch.where(total == 0.0, 1.0, total)
    lse = top + torch.log(total)
    # back to the tokens' rows
    t = torch.arange(s["q"].shape[0], device="cuda")
    r = torch.searchsorted(s["starts"][1:].contiguous(), t.to(torch.int32), right=True)
    i = t - s["starts"][r]

    def rows(x):
        return x.unflatten(2, (most, group)).permute(0, 2, 1, 3, 4)[r, i].flatten(1, 2)

    return {"out": rows(out).to(dtype), "lse": rows(lse).squeeze(-1)}


# ---------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------
def _buffer(s, name, *shape, dtype=torch.uint8):
    """Outputs and workspaces, which a program keeps from step to step."""
    if name not in s:
        s[name] = torch.empty(shape, dtype=dtype, device="cuda")
    return s[name]


def _own_plan(case, s, B):
    L, stream = B.lib(), torch.cuda.current_stream().cuda_stream
    requests, tokens, i32 = case["requests"], s["tokens"], torch.int32
    if "work" not in s:
        _buffer(s, "work", B.workspace("bsq_kv4_plan_workspace", requests))
    out = {"starts": _buffer(s, "o_starts", requests + 1, dtype=i32), "lengths": _buffer(s, "o_lengths", requests, dtype=i32),
           "table": s["table"], "left": _buffer(s, "o_left", 2, dtype=i32),
           "requests": _buffer(s, "o_requests", tokens, dtype=i32), "positions": _buffer(s, "o_positions", tokens, dtype=i32),
           "slots": _buffer(s, "o_slots", tokens, dtype=i32)}
    B.check(L.bsq_kv4_plan(s["lengths"].data_ptr(), s["new"].data_ptr(), requests, s["table"].data_ptr(),
                           s["table"].shape[1], case["page"], s["free"].data_ptr(), s["pages"], s["count"].data_ptr(),
                           out["lengths"].data_ptr(), out["left"].data_ptr(), out["starts"].data_ptr(), tokens,
                           out["requests"].data_ptr(), out["positions"].data_ptr(), out["slots"].data_ptr(),
                           s["work"].data_ptr(), s["work"].numel(), stream), "kv4 plan")
    return out


def _the_rope(s, B, dims, interleaved):
    if "rope" not in s:
        s["rope"] = B.Rope(s["frequencies"].data_ptr(), dims, int(interleaved), s["factor"])
    return s["rope"]


def _own_rope(case, s, B):
    L, stream, (t, dtype, _) = B.lib(), torch.cuda.current_stream().cuda_stream, _TYPES[case["type"]]
    tokens, width, rope = case["tokens"], case["heads"] * case["dim"], _the_rope(s, B, case["dims"], case["interleaved"])
    out = {"out": _buffer(s, "out", tokens, width, dtype=dtype)}
    B.check(L.bsq_rope(rope, s["positions"].data_ptr(), s["x"].data_ptr(), t, tokens, case["heads"], case["dim"],
                       width + case["pad"], 0, out["out"].data_ptr(), width, stream), "rope")
    if case["train"]:
        out["dx"] = _buffer(s, "dx", tokens, width, dtype=dtype)
        B.check(L.bsq_rope(rope, s["positions"].data_ptr(), s["d_out"].data_ptr(), t, tokens, case["heads"], case["dim"],
                           width, 1, out["dx"].data_ptr(), width, stream), "rope backward")
    return out


def _the_cache(s, B, case, buffer):
    if "handle" not in s:
        s["handle"] = B.Kv4Pages(buffer.data_ptr(), s["pages"], case["page"], case["heads"], case["dim"])
    return s["handle"]


def _own_append(case, s, B):
    L, stream, (t, dtype, size) = B.lib(), torch.cuda.current_stream().cuda_stream, _TYPES[case["type"]]
    tokens, queries, heads, dim, x = case["tokens"], case["queries"], case["heads"], case["dim"], s["x"]
    if "pool" not in s:
        _buffer(s, "pool", L.bsq_kv4_cache_bytes(s["pages"], case["page"], heads, dim))
    cache = _the_cache(s, B, case, s["pool"])
    out = {n: _buffer(s, n, tokens, (queries if n == "q" else heads) * dim, dtype=dtype) for n in "qkv"}
    row, keys = x.shape[1], x.data_ptr() + queries * dim * size
    B.check(L.bsq_kv4_append(cache, _the_rope(s, B, dim, case["interleaved"]), s["positions"].data_ptr(),
                             s["slots"].data_ptr(), x.shape[0], t, x.data_ptr(), queries, row, out["q"].data_ptr(),
                             queries * dim, keys, row, keys + heads * dim * size, row, stream), "kv4 append")
    B.check(L.bsq_kv4_read(cache, s["slots"].data_ptr(), tokens, t, out["k"].data_ptr(), heads * dim, out["v"].data_ptr(),
                           heads * dim, stream), "kv4 read")
    return out


def _own_attention(case, s, B):
    L, stream, q = B.lib(), torch.cuda.current_stream().cuda_stream, s["q"]
    (o, dtype, _), tokens, queries, dim = _TYPES[case["out"]], q.shape[0], case["queries"], case["dim"]
    cache, requests, width = _the_cache(s, B, case, s["cache"]), case["requests"], s["table"].shape[1]
    most = case["new"] if case["chunks"] else 1
    if "work" not in s:
        _buffer(s, "work", B.workspace("bsq_kv4_attention_workspace", cache, width, requests, tokens, most, queries))
    out = {"out": _buffer(s, "out", tokens, queries, dim, dtype=dtype),
           "lse": _buffer(s, "lse", tokens, queries, dtype=torch.float32)}
    B.check(L.bsq_kv4_attention(cache, s["table"].data_ptr(), width, s["lengths"].data_ptr(), s["starts"].data_ptr(),
                                requests, q.data_ptr(), _TYPES[case["type"]][0], tokens, most, queries, queries * dim,
                                s["scale"], 1, case["window"], out["out"].data_ptr(), o, queries * dim,
                                out["lse"].data_ptr(), s["work"].data_ptr(), s["work"].numel(), stream), "kv4 attention")
    return out


def run(state):
    kind = state["case"]["kind"]
    if own:
        import bitsqz_amd as B

        form = {"plan": _own_plan, "rope": _own_rope, "append": _own_append, "attention": _own_attention}[kind]
        return form(state["case"], state, B)
    form = {"plan": _plain_plan, "rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[kind]
    return form(state["case"], state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] in ("plan", "attention"):
        pairs, page = _lengths(case), case["page"]
    if case["kind"] == "plan":
        total = sum(max(m, 0) for _, m in pairs)
        moved = sum(_pages(p + m, page) - _pages(p, page) if m >= 0 else _pages(p, page) for p, m in pairs)
        return {"bytes": 16 * len(pairs) + 12 * total + 8 * moved, "flops": 0}
    size = _TYPES[case["type"]][2]
    if case["kind"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"] * (2 if case["train"] else 1)
        return {"bytes": 2 * values * size + 4 * case["tokens"], "flops": 6 * values * case["dims"] / case["dim"] / 2}
    heads, dim = case["heads"], case["dim"]
    token = 17 * -(-dim // 32) * heads * 2  # bytes of one in the cache
    if case["kind"] == "append":
        values = case["tokens"] * dim
        return {"bytes": values * size * (2 * case["queries"] + 4 * heads) + 2 * case["tokens"] * token + 8 * case["tokens"],
                "flops": 3 * values * (case["queries"] + heads)}
    window, seen, held = case["window"], 0, 0
    for p, m in pairs:
        if window and p + m > window:
            # keys that some query sees, and pairs of a query and a key
            held += min(p + m, window + m - 1)
            seen += sum(min(p + i + 1, window) for i in range(m))
        else:
            held += p + m
            seen += m * p + m * (m + 1) // 2
    tokens = sum(m for _, m in pairs)
    b = held * token + tokens * case["queries"] * (dim * (size + _TYPES[case["out"]][2]) + 4)
    return {"bytes": b + 4 * sum(_pages(p + m, page) for p, m in pairs), "flops": 4 * seen * case["queries"] * dim}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _two_to(exponent):
    """FP64 powers of two, from their bits."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _mx4(x):
    """FP64 x through MX4 along its last axis."""
    dim = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -dim % 32)).reshape(*x.shape[:-1], -1, 32)
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
    return (level * v.sign() * _two_to(exponent)).reshape(*x.shape[:-2], -1)[..., :dim]


def _complex_turn(x, s, dims, interleaved, sign=1.0):
    """Pairs as complex numbers, times factor e^(i angle)."""
    x = x.double()
    head, rest = x[..., :dims], x[..., dims:]
    z = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = sign * s["positions"][: x.shape[0]].double().outer(s["frequencies"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None]
    y = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, rest), -1)


def _levels(codes, scales, dim):
    """FP64 values of one head's codes (tokens x bytes) and scales (tokens x blocks)."""
    levels = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), dtype=torch.float64, device=codes.device)
    nibbles = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.uint8, device=codes.device)
    nibbles[..., 0::2] = codes % 16
    nibbles[..., 1::2] = codes // 16
    v = levels[(nibbles % 8).long()] * (1.0 - 2.0 * (nibbles >= 8))
    return (v * _two_to(scales.to(torch.int64) - 127).repeat_interleave(32, -1))[..., :dim]


def _exact_attention(case, s):
    page, dim, blocks, heads = case["page"], case["dim"], -(-case["dim"] // 32), case["heads"]
    group, tokens = case["queries"] // heads, s["q"].shape[0]
    out = torch.zeros(tokens, case["queries"], dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, case["queries"]), -math.inf, dtype=torch.float64, device="cuda")
    lengths, starts = s["lengths"].tolist(), s["starts"].tolist()
    row = 16 * blocks * page
    t = torch.arange(page, device="cuda")
    # a page's scale bytes: where those of its tokens are
    where = (t // 16 * 16 * blocks + t % 4 * 4 * blocks + t % 16 // 4)[:, None] + 4 * torch.arange(blocks, device="cuda")
    for r, n in enumerate(lengths):
        mine = s["cache"][s["table"][r, : _pages(n, page)].long()]  # pages x heads x bytes
        position = torch.arange(starts[r], starts[r + 1], device="cuda") - starts[r + 1] + n
        for h in range(heads):
            b = mine[:, h]
            k = _levels(b[:, :row].reshape(-1, 16 * blocks), b[:, 2 * row:][:, where].reshape(-1, blocks), dim)[:n]
            v = _levels(b[:, row: 2 * row].reshape(-1, 16 * blocks),
                        b[:, 2 * row + page * blocks:][:, where].reshape(-1, blocks), dim)[:n]
            key = torch.arange(n, device="cuda")
            hidden = key > position[:, None]
            if case["window"]:
                hidden |= key + case["window"] <= position[:, None]
            for head in range(h * group, (h + 1) * group):
                score = s["q"][starts[r]: starts[r + 1], head].double() @ k.T * s["scale"]
                score.masked_fill_(hidden, -math.inf)
                lse[starts[r]: starts[r + 1], head] = torch.logsumexp(score, 1)
                out[starts[r]: starts[r + 1], head] = torch.softmax(score, 1) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    if case["kind"] == "append":
        q, k, v = _parts(case, s["x"])
        # what is packed are the turned keys in their own type
        k = _complex_turn(k, s, case["dim"], case["interleaved"]).to(s["x"].dtype).double()
        return {"q": _complex_turn(q, s, case["dim"], case["interleaved"]).flatten(1), "k": _mx4(k).flatten(1),
                "v": _mx4(v.double()).flatten(1)}
    shape = (case["tokens"], case["heads"], case["dim"])
    got = {"out": _complex_turn(s["x"].reshape(shape), s, case["dims"], case["interleaved"]).flatten(1)}
    if case["train"]:
        got["dx"] = _complex_turn(s["d_out"].reshape(shape), s, case["dims"], case["interleaved"], -1.0).flatten(1)
    return got
