"""The paged MX4 cache (csrc/kv4.hip, csrc/kv4_attention.hip): its bookkeeping,
rotary positions, append, read and attention against their definitions in 64 bits
(_kv4ref.py).

The plan's whole numbers and the cache's bytes are defined bit by bit.  Turned
values are rounded through FP32: half a unit in the last place of each (2^-24 and
the type's), and 2^-40 of the pair for angles (2^21 positions times FP64's 2^-53,
and sine and cosine).  Products of FP32 values are FP64; of 16-bit ones FP32: sine
and cosine rounded, one product rounded and a fused sum, 3 2^-24 of the pair's
largest (sine plus cosine up to sqrt 2): 2^-22.  Attention is held to attention_bound,
plus the output type's rounding."""
import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_mx4 import ROUNDING, TYPES, stored, values

pytestmark = pytest.mark.gpu

LOWEST = {B.TYPE_F32: 2.0**-149, B.TYPE_BF16: 2.0**-133, B.TYPE_F16: 2.0**-24}  # smallest steps
DEPTH = {B.TYPE_F32: 3, B.TYPE_BF16: 1, B.TYPE_F16: 2}


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def run_plan(lengths, new, table, page, free, count, pages, tokens, alias=False, requests_out=True):
    L = B.lib()
    requests, width = table.shape
    dev = {n: B.DeviceBuffer.from_array(np.ascontiguousarray(v, np.int32)) for n, v in
           dict(lengths=lengths, new=new, table=table, free=free, count=[count, 0]).items()}
    out, left = (dev["lengths"], dev["count"]) if alias else (B.DeviceBuffer(4 * requests), B.DeviceBuffer(8))
    starts, places = B.DeviceBuffer(4 * (requests + 1)), [B.DeviceBuffer(4 * tokens) for _ in range(3)]
    work = B.DeviceBuffer(B.workspace("bsq_kv4_plan_workspace", requests))
    B.check(L.bsq_kv4_plan(dev["lengths"].ptr, dev["new"].ptr, requests, dev["table"].ptr, width, page, dev["free"].ptr,
                           pages, dev["count"].ptr, out.ptr, left.ptr, starts.ptr, tokens,
                           places[0].ptr if requests_out else None, places[1].ptr, places[2].ptr, work.ptr, work.nbytes,
                           None), "plan")
    B.check(L.bsq_stream_synchronize(None), "sync")
    got = left.download(np.int32, 2)
    return {"starts": starts.download(np.int32, requests + 1), "lengths": out.download(np.int32, requests),
            "table": dev["table"].download(np.int32, requests * width).reshape(requests, width),
            "free": dev["free"].download(np.int32, len(free)), "left": got[0], "unserved": got[1],
            "requests": places[0].download(np.int32, tokens), "positions": places[1].download(np.int32, tokens),
            "slots": places[2].download(np.int32, tokens)}


def check_plan(lengths, new, table, page, free, count, pages, tokens, **k):
    want = K.plan(lengths, new, np.asarray(table), page, free, count, pages, tokens)
    got = run_plan(lengths, new, np.asarray(table), page, free, count, pages, tokens, **k)
    for name, v in want.items():
        if name == "requests" and not k.get("requests_out", True):
            continue
        g = got[name][: len(v)] if name == "free" else got[name]
        assert np.array_equal(g, v), name
    return got


def scene(rng, requests, page, width, spare, most=40, ended=0.1):
    """Requests that hold pages of a shuffled pool, and new tokens."""
    lengths = rng.integers(0, width * page // 2 + 1, requests)
    new = rng.choice([0, 1, 1, 1, 2, most], requests)
    new[rng.random(requests) < ended] = -1
    new = np.where((new > 0) & (lengths + new > width * page), 1, new)
    held = -(-lengths // page)
    need = np.where(new < 0, 0, -(-(lengths + np.maximum(new, 0)) // page) - held)
    count = max(0, int(need.sum() - held[new < 0].sum()) + spare)
    pages = int(held.sum()) + count
    order = rng.permutation(pages)
    table = np.full((requests, width), -1)
    table[np.arange(width) < held[:, None]] = order[: held.sum()]
    free = np.full(max(pages, 1), -7)
    free[:count] = order[held.sum():]
    return lengths, new, table, page, free, count, pages, int(np.maximum(new, 0).sum())


@pytest.mark.parametrize("requests,page,width,spare,extra", [
    (1, 16, 4, 3, 0), (3, 32, 5, 0, 5), (64, 16, 40, 20, 64), (65, 256, 3, -2, 0), (1000, 16, 30, 100, 7), (1024, 64, 9, -30, 100),
    (1025, 16, 20, 5, 33), (3000, 32, 12, -400, 0), (16384, 16, 6, 1000, 100),
])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(requests, page, width, spare, extra, alias):
    rng = np.random.default_rng(requests + page)
    lengths, new, table, page, free, count, pages, tokens = scene(rng, requests, page, width, spare)
    check_plan(lengths, new, table, page, free, count, pages, tokens + extra, alias=alias)


def test_plan_one_and_two_launches_agree_at_the_border():
    rng = np.random.default_rng(9)
    lengths, new, table, page, free, count, pages, tokens = scene(rng, 500, 16, 200, 400, most=300)
    assert tokens > 4096
    for places in (4096, 4097, tokens, tokens + 5):  # the first are too few for all
        check_plan(lengths, new, table, page, free, count, pages, places)


def test_plan_without_requests_or_tokens():
    got = check_plan([], [], np.zeros((0, 3), int), 16, np.arange(5), 5, 5, 4)
    assert got["left"] == 5 and (got["slots"] == -1).all()
    check_plan([40, 7], [0, -1], np.array([[2, 1, 4], [3, -1, -1]]), 16, np.array([0, 9, 9, 9, 9]), 1, 5, 0)
    check_plan([40, 7], [1, -1], np.array([[2, 1, 4], [3, -1, -1]]), 16, np.array([0, 9, 9, 9, 9]), 1, 5, 1, requests_out=False)


def test_plan_refuses_single_requests():
    # a row that is too short, a stack that runs out, places that run out
    table = np.full((4, 2), -1)
    table[0, 0], table[3, 0] = 5, 3
    free = np.array([0, 1, 2, 4, -1, -1, -1])
    got = check_plan([16, 0, 0, 10], [16, 40, 20, 2], table, 16, free, 4, 7, 100)
    assert got["unserved"] == 1 and (got["slots"][16:56] == -1).all() and got["lengths"][1] == 0
    got = check_plan([16, 0, 0, 10], [16, 30, 20, 2], table, 16, free, 2, 7, 100)
    assert got["unserved"] == 2 and got["slots"][66] == 3 * 16 + 10  # needs no page
    got = check_plan([16, 0, 0, 10], [16, 10, 20, 2], table, 16, free, 4, 7, 30)
    assert got["unserved"] == 2 and got["starts"][-1] == 30


def test_plan_lengths_and_counts_out_of_range():
    table = np.array([[0, 1], [2, -1], [3, 4]])
    free = np.array([5, 6, 7, -1, -1, -1, -1, -1])
    check_plan([20, -5, 32], [3, 4, -1], table, 16, free, 3, 8, 9)
    check_plan([20, 2**31 - 1, 32], [3, 2**31 - 1, 0], table, 16, free, 3, 8, 9)
    check_plan([20, 2**31 - 1, 32], [3, -2**31, 0], table, 16, free, 3, 8, 9)  # gives its row
    check_plan([20, 3, 4], [30, 1, 1], np.repeat(table, 3, 1), 16, free, -4, 8, 40)
    check_plan([20, 3, 4], [1, 1, 1], table, 16, free, 2**31 - 1, 8, 3)
    check_plan([20, 3, 4], [1, 1, 1], np.array([[0, 99], [-3, 1], [4, 4]]), 16, free, 3, 8, 3)  # numbers outside


# ---------------------------------------------------------------------------
# rope
# ---------------------------------------------------------------------------
def turned_bound(want, x, type):
    """What turned values may be off by, from their pairs' magnitudes."""
    products = 2.0**-40 if type == B.TYPE_F32 else 2.0**-22
    return (ROUNDING[type] + 2.0**-24) * np.abs(want) + products * np.abs(x).max() + LOWEST[type]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tokens,heads,dim,dims,interleaved", [
    (1, 1, 2, 2, False), (3, 2, 64, 64, False), (5, 3, 64, 64, True), (17, 40, 128, 128, False), (9, 5, 80, 80, False),
    (9, 5, 80, 36, True), (7, 3, 100, 50, False), (7, 3, 33, 18, True), (4, 2, 256, 256, False), (2100, 1, 8, 6, False),
    (5000, 3, 16, 16, True), (300, 65, 48, 20, False),
])
def test_rope(type, tokens, heads, dim, dims, interleaved):
    rng = np.random.default_rng(tokens + dim + dims)
    raw, x = stored(rng.standard_normal((tokens, heads, dim)), type)
    positions = rng.integers(-1, 1 << rng.integers(1, 22), tokens).astype(np.int32)
    f, _ = B.rope_frequencies(dims, 10000.0)
    turn = B.Turn(f, 1.25, interleaved)
    for back in (False, True):
        got = values(B.rope(raw, positions, turn, type, back), type)
        want = K.turned(x, positions, f, 1.25, interleaved, back)
        assert (np.abs(got - want) <= turned_bound(want, 1.25 * x, type)).all()
        away = np.ones(got.shape, bool)
        away[..., :dims] = False
        away[positions < 0] = True
        assert np.array_equal(got[away], x[away])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    # against the formula's transpose (above) and against differences: the map is
    # linear, so a step of any size gives its derivative
    rng = np.random.default_rng(2)
    x, d = (rng.standard_normal((6, 3, 24)).astype(np.float32) for _ in range(2))
    positions = rng.integers(0, 100000, 6).astype(np.int32)
    turn = B.Turn(B.rope_frequencies(20, 10000.0)[0], 0.75, interleaved)
    dx = B.rope(d, positions, turn, back=True)
    y = B.rope(x, positions, turn).astype(np.float64)
    for at in [(0, 0, 0), (1, 2, 5), (3, 1, 11), (5, 0, 19), (2, 2, 20), (4, 1, 23)]:
        moved = x.copy()
        moved[at] += 1.0
        slope = ((B.rope(moved, positions, turn).astype(np.float64) - y) * d).sum()
        # each y is off by 2^-23 of itself, and x + 1 is rounded
        assert abs(slope - dx[at]) <= 2.0**-21 * np.abs(d).max() * np.abs(y).max() * 4


def test_rope_strides_and_rows_between():
    L, rng = B.lib(), np.random.default_rng(5)
    tokens, heads, dim, ldx, ldo = 37, 3, 20, 67, 71
    turn = B.Turn(B.rope_frequencies(16, 500.0)[0], 1.0, False)
    x, positions = rng.standard_normal((tokens, ldx)).astype(np.float32), rng.integers(-1, 1000, tokens).astype(np.int32)
    before = rng.standard_normal((tokens, ldo)).astype(np.float32)
    d, p, out = B.DeviceBuffer.from_array(x), B.DeviceBuffer.from_array(positions), B.DeviceBuffer.from_array(before)
    B.check(L.bsq_rope(turn.rope, p.ptr, d.ptr, 0, tokens, heads, dim, ldx, 0, out.ptr, ldo, None), "rope")
    B.check(L.bsq_stream_synchronize(None), "sync")
    got = out.download(np.float32, before.size).reshape(before.shape)
    want = K.turned(x[:, : heads * dim].reshape(tokens, heads, dim), positions, B.rope_frequencies(16, 500.0)[0]).reshape(tokens, -1)
    real = positions >= 0
    assert np.array_equal(got[:, heads * dim:], before[:, heads * dim:]) and np.array_equal(got[~real], before[~real])
    assert (np.abs(got[real, : heads * dim] - want[real]) <= turned_bound(want, x, B.TYPE_F32)[real]).all()


def test_rope_far_positions():
    # 2^31 - 1 positions on, angles of 2^31 radians: FP64's product is the definition
    x = np.ones((2, 1, 4), np.float32)
    positions = np.array([2**31 - 1, 123456789], np.int32)
    f = np.array([1.0, 0.9])
    got = B.rope(x, positions, B.Turn(f))
    want = K.turned(x, positions, f)
    assert np.abs(got - want).max() <= 2.0**-23 + 2.0**-40


# ---------------------------------------------------------------------------
# append, read
# ---------------------------------------------------------------------------
def appended(pages, page, heads, dim, slots, k, v, type, turn=None, positions=None, q=None, before=None):
    """The cache's bytes after the call, as K.Cache, and the queries."""
    L = B.lib()
    c = K.Cache(pages, page, heads, dim)
    if before is not None:
        c.bytes[:] = before
    buffer = B.DeviceBuffer.from_array(c.bytes)
    assert buffer.nbytes == L.bsq_kv4_cache_bytes(pages, page, heads, dim)
    handle = B.Kv4Pages(buffer.value, pages, page, heads, dim)
    n, row = len(slots), heads * dim
    dev = [B.DeviceBuffer.from_array(np.ascontiguousarray(a)) for a in (k, v, np.asarray(slots, np.int32))]
    p = B.DeviceBuffer.from_array(np.asarray(positions, np.int32)) if positions is not None else None
    dq = B.DeviceBuffer.from_array(q) if q is not None else None
    out = B.DeviceBuffer(q.nbytes) if q is not None else None
    wide = q.shape[1] if q is not None else 0
    if out is not None:
        out.zero()
    B.check(L.bsq_kv4_append(handle, turn.rope if turn else None, p.ptr if p else None, dev[2].ptr, n, type,
                             dq.ptr if dq else None, wide, wide * dim, out.ptr if out else None, wide * dim, dev[0].ptr,
                             row, dev[1].ptr, row, None), "append")
    B.check(L.bsq_stream_synchronize(None), "sync")
    c.bytes[:] = buffer.download(np.uint8, buffer.nbytes).reshape(c.bytes.shape)
    c.buffer, c.handle = buffer, handle
    return c, out.download(q.dtype, q.size).reshape(q.shape) if q is not None else None


SHAPES = [(1, 16, 1, 1, 1), (5, 16, 2, 64, 33), (3, 32, 8, 128, 70), (4, 64, 3, 80, 41), (2, 256, 1, 96, 300), (9, 16, 5, 33, 20),
          (3, 128, 2, 256, 17), (40, 16, 1, 8, 600), (3, 16, 4, 160, 30), (3, 16, 1, 200, 13)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("pages,page,heads,dim,tokens", SHAPES)
def test_append_and_read(type, pages, page, heads, dim, tokens):
    rng = np.random.default_rng(dim + tokens)
    (k, k64), (v, v64) = (stored(rng.standard_normal((tokens, heads, dim)) * np.exp(rng.standard_normal((tokens, heads, 1))), type) for _ in range(2))
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots = np.concatenate((slots, np.full(tokens - len(slots), -1)))
    slots[rng.random(tokens) < 0.1] = -1
    if tokens > 4:
        slots[2], slots[3] = pages * page, 2**31 - 1  # outside
    before = rng.integers(0, 255, (pages, heads, 34 * -(-dim // 32) * page)).astype(np.uint8)
    c, _ = appended(pages, page, heads, dim, slots, k, v, type, before=before)
    want = K.Cache(pages, page, heads, dim)
    want.bytes[:] = before
    for t in range(tokens):
        want.put(slots[t], k64[t], v64[t])
    assert np.array_equal(c.bytes, want.bytes)

    out = B.Kv4Cache.__new__(B.Kv4Cache)
    out.heads, out.dim, out.cache = heads, dim, c.handle
    got = out.read(slots, type)
    for which in (0, 1):
        for t in range(tokens):
            for h in range(heads):
                inside = 0 <= slots[t] < pages * page
                w = want.get(int(slots[t]), h, which) if inside else np.zeros(dim)
                assert np.array_equal(values(got[which][t, h], type), stored(w, type)[1])


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("heads,queries,dim,dims,interleaved,tokens", [
    (2, 4, 64, 64, False, 21), (1, 3, 128, 128, True, 40), (3, 6, 80, 40, False, 9), (2, 2, 33, 22, True, 15), (8, 32, 128, 128, False, 37),
    (1, 1, 256, 256, False, 7), (40, 40, 96, 96, False, 5), (1, 2, 16, 6, True, 3000),
])
def test_append_turned(type, heads, queries, dim, dims, interleaved, tokens):
    # a key is turned in 64 bits, rounded through FP32 to its type, then packed:
    # bytes agree but where sine and cosine's 2^-53 decides
    rng = np.random.default_rng(dim + tokens + heads)
    (k, k64), (v, v64) = (stored(rng.standard_normal((tokens, heads, dim)), type) for _ in range(2))
    q, q64 = stored(rng.standard_normal((tokens, queries, dim)), type)
    pages, page = tokens // 16 + 3, 16
    slots = rng.permutation(pages * page)[:tokens]
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    positions[tokens // 2] = -1
    f, _ = B.rope_frequencies(dims, 10000.0)
    turn = B.Turn(f, 1.1, interleaved)
    turn.rope.factor = 1.1
    factor = float(np.float32(1.1))
    c, got = appended(pages, page, heads, dim, slots, k, v, type, turn, positions, q)
    want = K.Cache(pages, page, heads, dim)
    k_want = stored(K.turned(k64, positions, f, factor, interleaved).astype(np.float32), type)[1]
    for t in range(tokens):
        if positions[t] >= 0:
            want.put(int(slots[t]), k_want[t], v64[t])
    assert np.array_equal(c.bytes, want.bytes)
    q_want = np.where((positions < 0)[:, None, None], 0.0, K.turned(q64, positions, f, factor, interleaved))
    assert (np.abs(values(got, type) - q_want) <= turned_bound(q_want, 1.1 * q64, type)).all()


def test_append_of_one_product_in_place():
    # queries, keys and values side by side, queries turned where they are
    L, rng = B.lib(), np.random.default_rng(8)
    tokens, queries, heads, dim = 50, 6, 2, 64
    raw, x = stored(rng.standard_normal((tokens, queries + 2 * heads, dim)), B.TYPE_BF16)
    c = B.Kv4Cache(6, 16, heads, dim, 1, 6)
    c.step([tokens])
    f, _ = B.rope_frequencies(dim)
    turn = B.Turn(f)
    d, row = B.DeviceBuffer.from_array(raw), (queries + 2 * heads) * dim
    at = d.value
    B.check(L.bsq_kv4_append(c.cache, turn.rope, c.positions.ptr, c.slots.ptr, tokens, 1, at, queries, row, at, row,
                             at + 2 * queries * dim, row, at + 2 * (queries + heads) * dim, row, None), "append")
    B.check(L.bsq_stream_synchronize(None), "sync")
    got = d.download(np.uint16, raw.size).reshape(raw.shape)
    assert np.array_equal(got[:, queries:], raw[:, queries:])
    positions = np.arange(tokens)
    want = K.turned(x[:, :queries], positions, f)
    assert (np.abs(values(got[:, :queries], B.TYPE_BF16) - want) <= turned_bound(want, x, B.TYPE_BF16)).all()
    k, v = c.read(c.slots.download(np.int32, tokens))
    assert np.array_equal(v, K.R.rounded(x[:, queries + heads:]))
    assert np.array_equal(k, K.R.rounded(stored(K.turned(x[:, queries: queries + heads], positions, f).astype(np.float32), B.TYPE_BF16)[1]))


def test_append_of_nan_and_infinity():
    k = np.ones((3, 1, 64), np.float32)
    v = np.ones((3, 1, 64), np.float32)
    k[0, 0, 5], k[1, 0, 40], v[2, 0, 1] = np.nan, np.inf, -np.inf
    c, _ = appended(1, 16, 1, 64, [0, 1, 2], k, v, B.TYPE_F32)
    want = K.Cache(1, 16, 1, 64)
    for t in range(3):
        want.put(t, k[t].astype(np.float64), v[t].astype(np.float64))
    assert np.array_equal(c.bytes, want.bytes) and (c.bytes == 255).sum() == 3


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def filled(rng, pages, page, heads, dim):
    """A cache whose every token is something, on the GPU too."""
    c = K.Cache(pages, page, heads, dim)
    n = pages * page
    (k, k64), (v, v64) = (stored(rng.standard_normal((n, heads, dim)) * np.exp(0.5 * rng.standard_normal((n, heads, 1))), B.TYPE_F32) for _ in range(2))
    for s in range(n):
        c.put(s, k64[s], v64[s])
    return c


def attend(c, table, lengths, counts, q, scale, type, out_type, causal=True, window=0, most=None, starts=True, extra=0, tokens=None):
    L = B.lib()
    requests, width = table.shape
    n, queries, dim = q.shape
    buffer = B.DeviceBuffer.from_array(c.bytes)
    handle = B.Kv4Pages(buffer.value, c.pages, c.page, c.heads, dim)
    dev = [B.DeviceBuffer.from_array(np.ascontiguousarray(a, np.int32)) for a in (table, lengths, np.concatenate(([0], np.cumsum(counts))))]
    row = queries * dim + extra
    padded = np.zeros((n, row), q.dtype)
    padded[:, : queries * dim] = q.reshape(n, -1)
    dq = B.DeviceBuffer.from_array(padded)
    t = B._TYPE_NUMPY[out_type]
    out, lse = B.DeviceBuffer.from_array(np.full((n, row), 7, t)), B.DeviceBuffer.from_array(np.full((n, queries), 7, np.float32))
    most = max(max(counts), 1) if most is None else most
    work = B.DeviceBuffer(B.workspace("bsq_kv4_attention_workspace", handle, width, requests, n, most, queries))
    work.upload(np.full(work.nbytes, 0xFF, np.uint8))  # NaN: nothing may hang on what it held
    for _ in range(2):
        B.check(L.bsq_kv4_attention(handle, dev[0].ptr, width, dev[1].ptr, dev[2].ptr if starts else None, requests, dq.ptr,
                                    type, n, most, queries, row, scale, int(causal), window, out.ptr, out_type, row, lse.ptr,
                                    work.ptr, work.nbytes, None), "attention")
        B.check(L.bsq_stream_synchronize(None), "sync")
        got = out.download(t, n * row).reshape(n, row)
        if _ == 0:
            first = got
    assert np.array_equal(first.view(np.uint8), got.view(np.uint8))  # the same from run to run
    assert (got[:, queries * dim:] == 7).all()
    return got[:, : queries * dim].reshape(n, queries, dim), lse.download(np.float32, n * queries).reshape(n, queries)


def check_attention(c, table, lengths, counts, q, scale, type=B.TYPE_BF16, out_type=None, causal=True, window=0, **k):
    out_type = type if out_type is None else out_type
    raw, q64 = stored(q, type)
    got, lse = attend(c, table, lengths, counts, raw, scale, type, out_type, causal, window, **k)
    got = values(got, out_type)
    depth = max(DEPTH[type], DEPTH[out_type])
    at = 0
    for r, n in enumerate(counts):
        mine = slice(at, at + n)
        at += n
        if n == 0:
            continue
        want, want_lse, of = K.attention(c, table[r], min(lengths[r], table.shape[1] * c.page), q64[mine], float(np.float32(scale)), causal, window)
        bound, lse_bound, _ = K.attention_bound(of, max(lengths[r], 1), q.shape[2], depth, 0)
        step = ROUNDING[out_type] * np.abs(want) + LOWEST[out_type]
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got[mine]), nan), r
        assert (np.abs(got[mine] - want)[~nan] <= (bound + step)[~nan]).all(), r
        none = want_lse == -np.inf
        assert np.array_equal(lse[mine] == -np.inf, none), r
        known = ~none & ~np.isnan(want_lse)
        assert np.array_equal(np.isnan(lse[mine]), np.isnan(want_lse)), r
        assert (np.abs(lse[mine][known] - want_lse[known]) <= lse_bound[known]).all(), r
    return got, lse, at


def tables(rng, c, lengths, width, spare=0):
    """Rows of different pages; places past a request's own hold nonsense."""
    order = rng.permutation(c.pages)
    table = rng.choice([-1, c.pages, 2**31 - 1, -2**31], (len(lengths), width))
    at = 0
    for r, n in enumerate(lengths):
        need = min(-(-n // c.page), width)
        table[r, :need] = order[np.arange(at, at + need) % c.pages]
        at += need
    return table


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("heads,group,dim,page", [(1, 1, 64, 16), (2, 4, 128, 16), (3, 5, 80, 32), (1, 8, 96, 64), (2, 16, 32, 16), (1, 17, 33, 16),
                                                  (2, 3, 256, 128), (1, 2, 160, 16), (1, 40, 8, 256), (1, 3, 200, 32)])
def test_single_tokens(type, heads, group, dim, page):
    rng = np.random.default_rng(heads * group + dim)
    c = filled(rng, max(3, 400 // page), page, heads, dim)
    lengths = [1, 15, 16, 17, 33, 0, 127, 128, 129, 300, 257, 31, 32]
    table = tables(rng, c, lengths, -(-320 // page))
    q = rng.standard_normal((len(lengths), heads * group, dim)) * 1.5
    check_attention(c, table, lengths, [1] * len(lengths), q, dim**-0.5, type)
    check_attention(c, table, lengths, [1] * len(lengths), q, dim**-0.5, type, starts=False)


@pytest.mark.parametrize("type,out_type", [(B.TYPE_BF16, B.TYPE_F32), (B.TYPE_F32, B.TYPE_BF16), (B.TYPE_F16, B.TYPE_F16), (B.TYPE_BF16, B.TYPE_F16),
                                           (B.TYPE_BF16, B.TYPE_BF16)])
@pytest.mark.parametrize("heads,group,dim,page,window", [(2, 2, 64, 16, 0), (1, 6, 128, 32, 0), (2, 1, 96, 16, 40), (1, 4, 48, 16, 7), (1, 3, 256, 64, 100),
                                                         (1, 32, 64, 16, 1)])
def test_chunks(type, out_type, heads, group, dim, page, window):
    # several queries a request, some more than keys, some none; a window
    rng = np.random.default_rng(dim + group)
    c = filled(rng, 640 // page, page, heads, dim)
    lengths, counts = [40, 5, 200, 0, 77, 33, 260, 1], [40, 9, 3, 2, 0, 1, 100, 1]
    table = tables(rng, c, lengths, -(-300 // page))
    q = rng.standard_normal((sum(counts), heads * group, dim))
    check_attention(c, table, lengths, counts, q, 0.11, type, out_type, window=window, extra=3)


@pytest.mark.parametrize("type", TYPES)
def test_not_causal(type):
    rng = np.random.default_rng(4)
    c = filled(rng, 20, 16, 2, 64)
    lengths, counts = [100, 3, 0, 64, 5], [7, 40, 2, 64, 0]
    q = rng.standard_normal((sum(counts), 4, 64))
    check_attention(c, tables(rng, c, lengths, 10), lengths, counts, q, 0.125, type, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0, 1e-30])
def test_scales(scale):
    rng = np.random.default_rng(6)
    c = filled(rng, 12, 16, 1, 64)
    lengths, counts = [150, 20], [1, 20]
    q = rng.standard_normal((21, 4, 64))
    check_attention(c, tables(rng, c, lengths, 10), lengths, counts, q, scale, B.TYPE_F32)


def test_scores_that_rise_and_fall():
    # the reference is raised again and again, or never after the first keys
    rng = np.random.default_rng(7)
    c = K.Cache(40, 16, 1, 32)
    for order in (1, -1):
        for s in range(640):
            k = np.full((1, 32), 0.01 * (s if order > 0 else 640 - s))
            c.put(s, k, rng.standard_normal((1, 32)))
        table = np.arange(40)[None]
        q = np.concatenate((np.full((1, 2, 32), 6.0), rng.standard_normal((1, 2, 32))), 1)
        check_attention(c, table, [640], [1], q, 1.0, B.TYPE_F32)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,count,past", [
    (1, 1, 64, 16, 65, 0), (2, 4, 128, 16, 50, 100), (1, 5, 96, 32, 90, 37), (1, 3, 256, 64, 60, 200), (1, 17, 33, 16, 9, 20),
    (2, 2, 160, 16, 64, 70), (1, 1, 200, 256, 129, 5), (1, 2, 8, 16, 150, 0), (1, 1, 192, 16, 100, -30), (1, 80, 64, 16, 3, 150),
])
def test_prompts(type, heads, group, dim, page, count, past):
    # alone (one kernel), beside others (two), in a window
    rng = np.random.default_rng(dim + count)
    c = filled(rng, max(4, 640 // page), page, heads, dim)
    length = count + past
    for lengths, counts in (([length], [count]), ([20, length, 0, 77], [1, count, 2, 70])):
        table = tables(rng, c, lengths, -(-320 // page))
        q = rng.standard_normal((sum(counts), heads * group, dim))
        check_attention(c, table, lengths, counts, q, dim**-0.5, type, extra=5)
        check_attention(c, table, lengths, counts, q, dim**-0.5, type, window=45)


@pytest.mark.parametrize("type", TYPES)
def test_prompts_not_causal(type):
    rng = np.random.default_rng(24)
    c = filled(rng, 20, 16, 2, 64)
    lengths, counts = [100, 0, 250], [90, 70, 3]
    q = rng.standard_normal((sum(counts), 4, 64))
    check_attention(c, tables(rng, c, lengths, 17), lengths, counts, q, 0.125, type, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales_of_prompts(scale):
    rng = np.random.default_rng(26)
    c = filled(rng, 12, 16, 1, 64)
    q = rng.standard_normal((80, 2, 64))
    check_attention(c, tables(rng, c, [150], 10), [150], [80], q, scale, B.TYPE_F32)


@pytest.mark.parametrize("window", [0, 1500])
def test_prompts_whose_keys_are_shared(window):
    # few tiles of queries over long contexts: workgroups share a tile's keys
    rng = np.random.default_rng(25)
    c = filled(rng, 320, 16, 1, 32)
    for lengths, counts in (([4800], [40]), ([4300, 2500, 3, 70], [50, 33, 3, 70])):
        table = np.array([rng.permutation(320) for _ in lengths])
        q = rng.standard_normal((sum(counts), 2, 32))
        for type in TYPES:
            check_attention(c, table, lengths, counts, q, 0.3, type, window=window)


def test_prompts_pages_out_of_range():
    rng = np.random.default_rng(28)
    c = filled(rng, 16, 16, 1, 64)
    lengths, counts = [200, 150], [80, 100]
    table = tables(rng, c, lengths, 14)
    table[0, 1], table[0, 3], table[0, 11], table[1, :] = -1, 16, 2**31 - 1, 99
    q = rng.standard_normal((sum(counts), 2, 64))
    got, lse, _ = check_attention(c, table, lengths, counts, q, 0.1, B.TYPE_F32)
    assert (got[80:] == 0).all() and (lse[80:] == -np.inf).all()


def test_prompts_nan_where_nobody_looks():
    rng = np.random.default_rng(29)
    for group, dim in ((1, 64), (3, 128), (1, 33), (2, 256)):
        for type in (B.TYPE_BF16, B.TYPE_F32):
            c = filled(rng, 16, 16, 1, dim)
            length, n = 190, 80  # queries at 110 .. 189
            table = np.array([rng.permutation(16)[:12]])
            slot = lambda j: int(table[0, j // 16]) * 16 + j % 16  # noqa: E731
            for j in range(length, 192):
                c.put(slot(j), np.full((1, dim), np.nan), np.full((1, dim), np.nan))
            v = c.get(slot(140), 0, 1).copy()
            v[3] = np.nan
            c.put(slot(140), c.get(slot(140), 0, 0)[None], v[None])
            q = rng.standard_normal((n, group, dim))
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type)
            assert np.isnan(got[30:, :, :32]).all() and np.isfinite(got[:30]).all() and np.isfinite(got[:, :, 32:]).all()
            check_attention(c, table, [length], [n], q, 0.1, type, window=20)
            k = c.get(slot(150), 0, 0).copy()
            k[0] = np.nan
            c.put(slot(150), k[None], c.get(slot(150), 0, 1)[None])
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type)
            assert np.isnan(lse[40:]).all() and np.isfinite(lse[:40]).all()
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type, window=20)
            assert np.isfinite(lse[:40]).all() and np.isnan(lse[40:60]).all() and np.isfinite(lse[60:]).all()


def test_long_request_over_all_workgroups():
    # one request whose keys many workgroups share, beside short ones
    rng = np.random.default_rng(11)
    c = filled(rng, 300, 16, 1, 32)
    lengths = [4700, 3, 60, 0, 4300, 900]
    table = np.array([rng.permutation(300) for _ in lengths])
    q = rng.standard_normal((len(lengths), 2, 32))
    for type in TYPES:
        check_attention(c, table, lengths, [1] * len(lengths), q, 0.3, type)
        check_attention(c, table, lengths, [1] * len(lengths), q, 0.3, type, window=1000)


def test_many_requests():
    rng = np.random.default_rng(12)
    c = filled(rng, 50, 16, 2, 32)
    for requests in (255, 256, 257, 1500):
        lengths = rng.integers(0, 90, requests)
        counts = rng.integers(0, 3, requests)
        table = rng.integers(0, 50, (requests, 6))
        q = rng.standard_normal((int(counts.sum()), 2, 32))
        check_attention(c, table, lengths, list(counts), q, 0.2, B.TYPE_BF16)


@pytest.mark.parametrize("window", [1, 319, 320, 2**31 - 1, 2**31, 2**32 - 1])
def test_windows_of_any_size(window):
    # as long as the table, longer than 31 bits; queries ahead of the first key
    rng = np.random.default_rng(30)
    c = filled(rng, 20, 16, 1, 64)
    lengths, counts = [320, 10, 300], [3, 40, 90]
    table = np.array([rng.permutation(20) for _ in lengths])
    q = rng.standard_normal((sum(counts), 2, 64))
    check_attention(c, table, lengths, counts, q, 0.1, B.TYPE_F32, window=window)


def test_rows_behind_and_past_most_are_left():
    rng = np.random.default_rng(13)
    c = filled(rng, 12, 16, 1, 64)
    lengths, counts = [30, 50], [3, 4]
    table = tables(rng, c, lengths, 5)
    q = rng.standard_normal((12, 2, 64))
    got, lse, at = check_attention(c, table, lengths, counts, q, 0.1, B.TYPE_F32)
    assert (got[at:] == 7).all() and (lse[at:] == 7).all()
    raw, q64 = stored(q, B.TYPE_F32)
    got, lse = attend(c, table, lengths, counts, raw, 0.1, 0, 0, most=3)
    assert (got[6:] == 7).all() and (lse[6:] == 7).all()
    want, want_lse, of = K.attention(c, table[1], 50, q64[3:7], float(np.float32(0.1)))
    assert np.abs(got[3:6] - want[:3]).max() < 1e-5  # as with all four


def test_pages_and_starts_out_of_range():
    # numbers outside the cache are not seen; lengths end with the table
    rng = np.random.default_rng(14)
    c = filled(rng, 12, 16, 1, 64)
    lengths, counts = [70, 500, 20], [2, 1, 6]
    table = tables(rng, c, [70, 96, 20], 6)
    table[0, 1], table[0, 3], table[1, 0], table[2, :] = -1, 12, 2**31 - 1, 99
    q = rng.standard_normal((9, 2, 64))
    got, lse, _ = check_attention(c, table, lengths, counts, q, 0.1, B.TYPE_F32)
    assert (got[3:] == 0).all() and (lse[3:] == -np.inf).all()
    raw, _ = stored(q, B.TYPE_F32)
    for starts in ([0, 4, 20, 30], [0, 8, 3, 3], [0, -1, 5, 2]):
        attend(c, table, lengths, np.diff([0] + starts[1:]), raw, 0.1, 0, 0, most=9)


def test_nan_where_nobody_looks():
    # NaN blocks of keys and values: those that a query does not see change nothing,
    # those that it sees make its channels NaN
    rng = np.random.default_rng(15)
    for group, dim in ((1, 64), (3, 128), (1, 33), (2, 256)):
        for type in TYPES:
            c = filled(rng, 12, 16, 1, dim)
            length, n = 100, 5
            table = np.array([rng.permutation(12)[:8]])
            slot = lambda j: int(table[0, j // 16]) * 16 + j % 16  # noqa: E731
            for j in range(length, 128):  # behind the last
                c.put(slot(j), np.full((1, dim), np.nan), np.full((1, dim), np.nan))
            v = c.get(slot(97), 0, 1).copy()
            v[3] = np.nan  # the first block, seen from the third query on
            c.put(slot(97), c.get(slot(97), 0, 0)[None], v[None])
            q = rng.standard_normal((n, group, dim))
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type)
            assert np.isnan(got[2:, :, :32]).all() and np.isfinite(got[:2]).all() and np.isfinite(got[:, :, 32:]).all()
            # a key, seen by the last query alone
            k = c.get(slot(99), 0, 0).copy()
            k[0] = np.nan
            c.put(slot(99), k[None], c.get(slot(99), 0, 1)[None])
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type)
            assert np.isnan(got[4]).all() and np.isnan(lse[4]).all() and np.isfinite(lse[:4]).all()
            # a window that has left a NaN key and a NaN value behind
            c.put(slot(53), np.full((1, dim), np.nan), np.full((1, dim), np.nan))
            got, lse, _ = check_attention(c, table, [length], [n], q, 0.1, type, window=44)
            assert np.isfinite(lse[3]).all() and np.isnan(lse[0]).all()


def test_queries_of_nan_and_infinity():
    rng = np.random.default_rng(16)
    c = filled(rng, 12, 16, 1, 64)
    q = rng.standard_normal((4, 2, 64)).astype(np.float32)
    q[0, 0, 3], q[2, 1, 60] = np.nan, np.inf
    raw, _ = stored(q, B.TYPE_BF16)
    got, lse = attend(c, tables(rng, c, [90], 6), [90], [4], raw, 0.1, 1, 1)
    bad = np.zeros((4, 2), bool)
    bad[0, 0] = bad[2, 1] = True
    assert np.array_equal(np.isnan(values(got, 1)).all(2), bad) and np.array_equal(np.isnan(lse), bad)


def test_offsets_past_32_bits():
    # a cache of 5 GiB, keys in its first and last pages
    L, rng = B.lib(), np.random.default_rng(17)
    heads, dim, page = 8, 128, 256
    each = L.bsq_kv4_cache_bytes(1, page, heads, dim)
    pages = 5 * 2**30 // each
    buffer = B.DeviceBuffer(pages * each)
    handle = B.Kv4Pages(buffer.value, pages, page, heads, dim)
    small = K.Cache(2, page, heads, dim)
    numbers = [0, pages - 1]
    tokens = 300
    (k, k64), (v, v64) = (stored(rng.standard_normal((tokens, heads, dim)), B.TYPE_BF16) for _ in range(2))
    slots = np.array([numbers[t // page] * page + t % page for t in range(tokens)], np.int32)
    dev = [B.DeviceBuffer.from_array(a) for a in (k, v, slots)]
    row = heads * dim
    B.check(L.bsq_kv4_append(handle, None, None, dev[2].ptr, tokens, 1, None, 0, 0, None, 0, dev[0].ptr, row, dev[1].ptr, row, None), "append")
    for t in range(tokens):
        small.put(t, k64[t], v64[t])
    table, q = np.array([numbers], np.int32), rng.standard_normal((1, heads, dim))
    raw, q64 = stored(q, B.TYPE_F32)
    dq, dt, dl = B.DeviceBuffer.from_array(raw), B.DeviceBuffer.from_array(table), B.DeviceBuffer.from_array(np.array([tokens], np.int32))
    out = B.DeviceBuffer(raw.nbytes)
    work = B.DeviceBuffer(B.workspace("bsq_kv4_attention_workspace", handle, 2, 1, 1, 1, heads))
    B.check(L.bsq_kv4_attention(handle, dt.ptr, 2, dl.ptr, None, 1, dq.ptr, 0, 1, 1, heads, row, 0.1, 1, 0, out.ptr, 0, row, None, work.ptr,
                                work.nbytes, None), "attention")
    B.check(L.bsq_stream_synchronize(None), "sync")
    got = out.download(np.float32, raw.size).reshape(raw.shape)
    want, _, of = K.attention(small, [0, 1], tokens, q64, float(np.float32(0.1)))
    bound, _, _ = K.attention_bound(of, tokens, dim, 3, 0)
    assert (np.abs(got - want) <= bound + 2.0**-24 * np.abs(want)).all()
    buffer.free()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_steps_of_a_server():
    # requests that come, go on and end, against caches kept on the host
    rng = np.random.default_rng(20)
    page, heads, queries, dim, requests = 16, 2, 6, 64, 5
    cache = B.Kv4Cache(24, page, heads, dim, requests, 8)
    f, factor = B.rope_frequencies(dim, 10000.0, B.ROPE_PARTS, 4.0, 32.0)
    turn = B.Turn(f, factor)
    held = [[] for _ in range(requests)]
    for new in ([20, 0, 7, 0, 0], [1, 33, 1, 0, 0], [1, 1, 1, 40, 0], [1, -1, 1, 1, 12], [16, 5, -1, 1, 1], [1, 1, 90, -1, 1], [1, 1, 1, 3, 1]):
        places = cache.step(new, tokens=int(np.maximum(new, 0).sum()) + 3)
        n = cache.tokens
        k, v, q = (stored(rng.standard_normal((n, h, dim)), B.TYPE_BF16)[0] for h in (heads, heads, queries))
        q = cache.append(k, v, q, turn, B.TYPE_BF16)
        out, lse = cache.attend(q, type=B.TYPE_BF16, out_type=B.TYPE_BF16)
        assert places["unserved"] == 0
        for r in range(requests):
            if new[r] < 0:
                held[r] = []
            for t in range(places["starts"][r], places["starts"][r + 1]):
                assert places["positions"][t] == len(held[r]) and places["requests"][t] == r
                turned = stored(K.turned(values(k[t:t + 1], 1), [len(held[r])], f, factor).astype(np.float32), 1)[1]
                held[r].append((turned[0], values(v[t], 1)))
        assert (places["slots"][-3:] == -1).all() and (out[-3:] == 0).all() and (lse[-3:] == -np.inf).all()
        for r in range(requests):
            mine = slice(places["starts"][r], places["starts"][r + 1])
            if mine.start == mine.stop:
                continue
            host = K.Cache(8, page, heads, dim)
            for t, (a, b) in enumerate(held[r]):
                host.put(t, a, b)
            want, _, of = K.attention(host, np.arange(8), len(held[r]), values(q[mine], 1), float(np.float32(dim**-0.5)))
            bound, _, _ = K.attention_bound(of, len(held[r]), dim, 1, 0)
            assert (np.abs(values(out[mine], 1) - want) <= bound + 2.0**-8 * np.abs(want)).all()
    assert places["left"] == 24 - sum(-(-len(h) // page) for h in held)
