"""Paths of the attention over the paged MX4 cache: prompts among many requests,
units of work of more than 32 keys, starts that overlap; and the example's steps
against their definitions."""
import os
import sys

import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_kv4 import check_attention, filled, turned_bound

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# requests, units, starts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type", [B.TYPE_BF16, B.TYPE_F32])
@pytest.mark.parametrize("requests,prompts", [
    (65, [0, 63, 64]), (64, [63]), (257, [5, 191, 192, 255, 256]), (256, [64, 255]), (1000, [0, 1, 2, 3, 511, 640, 998, 999]),
])
def test_prompts_among_many_requests(type, requests, prompts):
    # a thread of the prompts' kernel looks through one request, or several
    rng = np.random.default_rng(requests)
    c = filled(rng, 40, 16, 1, 32)
    lengths, counts = rng.integers(0, 90, requests), rng.integers(0, 3, requests)
    for i, r in enumerate(prompts):
        counts[r] = 65 + 33 * i  # 1 to 3 tiles
        lengths[r] = counts[r] + rng.integers(-20, 200)
    table = rng.integers(0, 40, (requests, 32))
    q = rng.standard_normal((int(counts.sum()), 1, 32))
    check_attention(c, table, list(lengths), list(counts), q, 0.2, type)
    check_attention(c, table, list(lengths), list(counts), q, 0.2, type, window=50)


@pytest.mark.parametrize("window", [0, 300])
def test_units_of_more_than_32_keys(window):
    # 3 requests x 2048 heads, rows of the table for 2^25 keys: with units of 32 keys
    # their number would not fit 31 bits
    rng = np.random.default_rng(40)
    heads, width = 2048, 1 << 21
    c = K.Cache(48, 16, heads, 8)
    codes = rng.integers(0, 256, (48, heads, 2 * 16, 16))
    codes[..., 4:] = 0  # the rows' padding
    c.bytes[:, :, :512] = codes.reshape(48, heads, 512)
    c.bytes[:, :, 512:] = rng.integers(125, 129, (48, heads, 32))
    table = np.full((3, width), -1, np.int32)
    for r in range(3):
        table[r, :48] = rng.permutation(48)
    lengths, counts = [740, 131, 40], [2, 1, 3]
    q = rng.standard_normal((6, heads, 8))
    check_attention(c, table, lengths, counts, q, 0.2, B.TYPE_BF16, window=window)


@pytest.mark.parametrize("starts,lengths,group,alone", [
    ([0, 8, 3, 9], [40, 50, 60], 2, {0: range(0, 3), 2: range(8, 9)}),
    ([0, 130, 10, 140], [200, 50, 170], 1, {0: range(0, 10), 2: range(130, 140)}),
])
def test_starts_that_overlap(starts, lengths, group, alone):
    # the second request has no query; rows of two requests may hold either's
    L, rng = B.lib(), np.random.default_rng(41)
    c = filled(rng, 14, 16, 1, 64)
    table = np.array([rng.permutation(14)[:13] for _ in lengths], np.int32)
    tokens = starts[-1]
    q = rng.standard_normal((tokens, group, 64)).astype(np.float32)
    pool = B.DeviceBuffer.from_array(c.bytes)
    handle = B.Kv4Pages(pool.value, c.pages, c.page, 1, 64)
    dev = [B.DeviceBuffer.from_array(np.ascontiguousarray(a, t)) for a, t in
           ((table, np.int32), (lengths, np.int32), (starts, np.int32), (q, np.float32))]
    out, lse = (B.DeviceBuffer.from_array(np.full(s, 7, np.float32)) for s in (q.shape, q.shape[:2]))
    work = B.DeviceBuffer(B.workspace("bsq_kv4_attention_workspace", handle, 13, 3, tokens, tokens, group))
    B.check(L.bsq_kv4_attention(handle, dev[0].ptr, 13, dev[1].ptr, dev[2].ptr, 3, dev[3].ptr, 0, tokens, tokens, group, group * 64,
                                0.1, 1, 0, out.ptr, 0, group * 64, lse.ptr, work.ptr, work.nbytes, None), "attention")
    B.check(L.bsq_stream_synchronize(None), "sync")
    out, lse = out.download(np.float32, q.size).reshape(q.shape), lse.download(np.float32, tokens * group).reshape(tokens, group)
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    for r, rows in alone.items():
        first, last = starts[r], starts[r + 1]
        want, want_lse, of = K.attention(c, table[r], lengths[r], q[first:last].astype(np.float64), float(np.float32(0.1)))
        bound, lse_bound, _ = K.attention_bound(of, lengths[r], 64, 3, 0)
        near = (np.abs(out[first:last] - want) <= bound + 2.0**-24 * np.abs(want)).all((1, 2))
        near &= (np.abs(lse[first:last] - want_lse) <= lse_bound).all(1)
        assert all(near[t - first] for t in rows)


# ---------------------------------------------------------------------------
# the example
# ---------------------------------------------------------------------------
class Followed(B.Kv4Cache):
    """A cache whose every step is compared with its definition in 64 bits."""
    steps = 0

    def __init__(self, pages, page, heads, dim, requests, width):
        super().__init__(pages, page, heads, dim, requests, width)
        self.host = K.Cache(pages, page, heads, dim)
        self.held = np.zeros(requests, int)

    def step(self, new, tokens=None):
        self.places = super().step(new, tokens)
        for r, n in enumerate(new):
            a, b = self.places["starts"][r], self.places["starts"][r + 1]
            assert b - a == max(n, 0) and self.places["positions"][a:b].tolist() == list(range(self.held[r], self.held[r] + b - a))
            self.held[r] = 0 if n < 0 else self.held[r] + n
        return self.places

    def append(self, k, v, q=None, turn=None, type=B.TYPE_F32):
        out = super().append(k, v, q, turn, type)
        f = turn.buffer.download(np.float64, turn.dims // 2)
        factor = float(turn.rope.factor)
        at, slots = self.places["positions"], self.places["slots"]
        turned = K.turned(k, at, f, factor).astype(np.float32).astype(np.float64)
        for t, s in enumerate(slots):
            self.host.put(int(s), turned[t], v[t].astype(np.float64))
        for which, got in enumerate(self.read(slots)):
            assert np.array_equal(got, self.host.values(which)[slots])
        want = K.turned(q, at, f, factor)
        assert (np.abs(out - want) <= turned_bound(want, factor * q, B.TYPE_F32)).all()
        return out

    def attend(self, q, **k):
        out, lse = super().attend(q, **k)
        table = self.table.download(np.int32, self.requests * self.width).reshape(self.requests, -1)
        for r in range(self.requests):
            a, b = self.places["starts"][r], self.places["starts"][r + 1]
            if a == b:
                continue
            want, want_lse, of = K.attention(self.host, table[r], self.held[r], q[a:b].astype(np.float64),
                                             float(np.float32(self.dim**-0.5)))
            bound, lse_bound, _ = K.attention_bound(of, self.held[r], self.dim, 3, 0)
            assert (np.abs(out[a:b] - want) <= bound + 2.0**-24 * np.abs(want)).all()
            assert (np.abs(lse[a:b] - want_lse) <= lse_bound).all()
        Followed.steps += 1
        return out, lse


def test_example_follows_the_definitions(monkeypatch):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import kv4_generate

    monkeypatch.setattr(kv4_generate.B, "Kv4Cache", Followed)
    Followed.steps = 0
    text, off = kv4_generate.generate(6)
    assert [len(t) for t in text] == [11, 37, 26]
    # prompts and steps, two layers; then two requests anew
    assert Followed.steps == 2 * (1 + 6) + 2 * 2
    assert off < 0.5  # the example's own limit: codes of activations next to a border may differ
