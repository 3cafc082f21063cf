"""What the entry points of the paged cache refuse (include/bitsqz_llm_c.h, group
7), without a GPU: the checks run before any device work.  Pointers that are
never reached are small integers of the right alignment."""
import ctypes as C

import numpy as np
import pytest

import bitsqz_amd as B

D = 4096  # a pointer that is not followed
NONE = 2**64 - 1


def refused(rc, word):
    msg = B.lib().bsq_last_error().decode()
    assert rc == 1 and word in msg, (rc, msg)


def cache(**k):
    a = dict(d_pages=D, pages=10, page=16, heads=2, dim=64)
    a.update(k)
    return B.Kv4Pages(*(a[n] for n, _ in B.Kv4Pages._fields_))


def rope(**k):
    a = dict(d_frequencies=D, dims=64, interleaved=0, factor=1.0)
    a.update(k)
    return B.Rope(*(a[n] for n, _ in B.Rope._fields_))


def test_cache_bytes():
    L = B.lib()
    for pages, page, heads, dim in ((1, 16, 1, 1), (7, 32, 3, 33), (5, 256, 8, 128), (2, 64, 1, 256), (0, 16, 1, 8)):
        assert L.bsq_kv4_cache_bytes(pages, page, heads, dim) == pages * heads * page * -(-dim // 32) * 34
    assert L.bsq_kv4_cache_bytes((2**31 - 1) // 16, 16, 65535, 256) == (2**31 - 1) // 16 * 65535 * 16 * 8 * 34
    for bad in ((1, 8, 1, 8), (1, 17, 1, 8), (1, 512, 1, 8), (1, 16, 0, 8), (1, 16, 65536, 8), (1, 16, 1, 0), (1, 16, 1, 257),
                (2**27, 16, 1, 8)):
        assert L.bsq_kv4_cache_bytes(*bad) == NONE and L.bsq_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(requests=16385), "requests"), (dict(page=24), "page"), (dict(pages=2**27), "pages"),
    (dict(requests=16384, width=2**17), "table"), (dict(requests=1, width=2**27), "too long"), (dict(tokens=2**31), "tokens"),
    (dict(count=None), "null"), (dict(left=None), "null"), (dict(starts=None), "null"), (dict(lengths=None), "null"),
    (dict(new=None), "null"), (dict(out=None), "null"), (dict(table=None), "table"), (dict(free=None), "stack"),
    (dict(positions=None), "output"), (dict(slots=None), "output"), (dict(work_bytes=0), "workspace"), (dict(work=None), "null"),
])
def test_plan(change, word):
    a = dict(lengths=D, new=D, requests=4, table=D, width=8, page=16, free=D, pages=40, count=D, out=D, left=D, starts=D,
             tokens=4, of=None, positions=D, slots=D, work=D, work_bytes=1 << 20, stream=None)
    a.update(change)
    refused(B.lib().bsq_kv4_plan(*a.values()), word)


def test_plan_workspace():
    assert B.lib().bsq_kv4_plan_workspace(16384) >= 4 * 16385
    assert B.lib().bsq_kv4_plan_workspace(16385) == NONE
    with pytest.raises(B.BsqError, match="16384"):
        B.workspace("bsq_kv4_plan_workspace", 20000)


@pytest.mark.parametrize("change,word", [
    (dict(rope=None), "null rope"), (dict(rope=rope(d_frequencies=None)), "frequencies"), (dict(rope=rope(d_frequencies=D + 4)), "unaligned"),
    (dict(rope=rope(dims=0)), "dims"), (dict(rope=rope(dims=33)), "dims"), (dict(rope=rope(dims=66)), "dims"),
    (dict(rope=rope(interleaved=2)), "interleaved"), (dict(rope=rope(factor=float("nan"))), "factor"),
    (dict(positions=None), "positions"), (dict(x=None), "null input"), (dict(out=None), "null output"), (dict(x=D + 1), "unaligned"),
    (dict(type=3), "type"), (dict(heads=65536), "heads"), (dict(dim=257, ldx=1 << 20, ldo=1 << 20), "heads of"), (dict(dim=0), "heads of"),
    (dict(ldx=127), "overlap"), (dict(ldo=127), "overlap"), (dict(tokens=2**31), "tokens"), (dict(ldx=2**29), "apart"),
    (dict(out=D, ldo=200), "overlaps"), (dict(out=D + 64), "overlaps"),
])
def test_rope(change, word):
    a = dict(rope=rope(), positions=D, x=D, type=1, tokens=4, heads=2, dim=64, ldx=128, back=0, out=1 << 20, ldo=128, stream=None)
    a.update(change)
    refused(B.lib().bsq_rope(*a.values()), word)


@pytest.mark.parametrize("args,word", [
    ((3, 1e4, 0, 1.0, 0.0), "even"), ((0, 1e4, 0, 1.0, 0.0), "even"), ((258, 1e4, 0, 1.0, 0.0), "even"), ((8, 1.0, 0, 1.0, 0.0), "base"),
    ((8, float("inf"), 0, 1.0, 0.0), "base"), ((8, float("nan"), 0, 1.0, 0.0), "base"), ((8, 1e4, 4, 1.0, 0.0), "scaling"),
    ((8, 1e4, 1, 0.5, 0.0), "stretch"), ((8, 1e4, 3, float("nan"), 9.0), "stretch"), ((2, 1e4, 2, 2.0, 0.0), "4 dims"),
    ((8, 1e4, 3, 2.0, 0.0), "length"),
])
def test_frequencies(args, word):
    with pytest.raises(B.BsqError, match=word):
        B.rope_frequencies(*args)
    f = C.c_float()
    refused(B.lib().bsq_rope_frequencies(8, 1e4, 0, 1.0, 0.0, None, C.byref(f)), "null")


def test_frequencies_values():
    i = np.arange(32)
    f = 1e4 ** (-2.0 * i / 64)
    for scaling, stretch, want in ((0, 9.0, f), (1, 4.0, f / 4), (2, 4.0, (1e4 * 4 ** (64 / 62)) ** (-2.0 * i / 64))):
        got, factor = B.rope_frequencies(64, 1e4, scaling, stretch, 100.0)
        np.testing.assert_allclose(got, want, rtol=1e-14)
        assert factor == 1.0
    got, factor = B.rope_frequencies(64, 1e4, 3, 8.0, 4096.0)
    assert factor == np.float32(1 + 0.1 * np.log(8.0))
    turns = 4096 * f / (2 * np.pi)
    assert np.allclose(got[turns > 34], f[turns > 34]) and np.allclose(got[turns < 0.9], f[turns < 0.9] / 8)
    between = (turns > 1.1) & (turns < 30)
    assert between.any() and ((got < f) & (got > f / 8))[between].all() and (np.diff(got) < 0).all()
    # a stretch of 1 changes nothing
    for scaling in (1, 2, 3):
        got, factor = B.rope_frequencies(64, 1e4, scaling, 1.0, 4096.0)
        np.testing.assert_allclose(got, f, rtol=1e-14)
        assert factor == 1.0


@pytest.mark.parametrize("change,word", [
    (dict(cache=None), "null cache"), (dict(cache=cache(d_pages=None)), "null cache"), (dict(cache=cache(d_pages=D + 8)), "aligned"),
    (dict(cache=cache(page=20)), "page"), (dict(cache=cache(dim=0)), "heads of"), (dict(cache=cache(dim=257)), "heads of"),
    (dict(cache=cache(heads=0)), "heads"), (dict(cache=cache(pages=0)), "null cache"), (dict(cache=cache(pages=2**27)), "pages"),
    (dict(type=-1), "type"), (dict(slots=None), "slots"), (dict(k=None), "keys"), (dict(v=None), "values"), (dict(k=D + 1), "unaligned"),
    (dict(q_out=None), "null output"), (dict(q=D + 1), "unaligned"), (dict(ldk=127), "overlap"), (dict(ldv=127), "overlap"), (dict(ldq=255), "overlap"),
    (dict(ldqo=255), "overlap"), (dict(q_out=D + 256), "overlaps"), (dict(rope=rope(), positions=None), "positions"),
    (dict(rope=rope(dims=66)), "dims"), (dict(tokens=2**31), "tokens"), (dict(q_heads=65536), "heads"),
])
def test_append(change, word):
    a = dict(cache=cache(), rope=rope(), positions=D, slots=D, tokens=4, type=1, q=D, q_heads=4, ldq=256, q_out=1 << 20, ldqo=256,
             k=D, ldk=128, v=D, ldv=128, stream=None)
    a.update(change)
    refused(B.lib().bsq_kv4_append(*a.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(cache=cache(page=0)), "page"), (dict(slots=None), "slots"), (dict(k=D + 1), "unaligned"), (dict(v=D + 1), "unaligned"), (dict(ldk=127), "overlap"),
    (dict(ldv=127), "overlap"), (dict(type=3), "type"),
])
def test_read(change, word):
    a = dict(cache=cache(), slots=D, tokens=4, type=1, k=D, ldk=128, v=D, ldv=128, stream=None)
    a.update(change)
    refused(B.lib().bsq_kv4_read(*a.values()), word)


def attention_args(**change):
    a = dict(cache=cache(), table=D, width=8, lengths=D, starts=D, requests=3, q=D, q_type=1, tokens=6, most=4, q_heads=4, ldq=256,
             scale=0.125, causal=1, window=0, out=1 << 20, out_type=1, ldo=256, lse=None, work=D, work_bytes=1 << 30, stream=None)
    a.update(change)
    return a.values()


@pytest.mark.parametrize("change,word", [
    (dict(cache=cache(page=0)), "page"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"), (dict(q_heads=65536), "65535"),
    (dict(tokens=2**31), "queries"), (dict(tokens=2**30, q_heads=64, ldq=1 << 20, ldo=1 << 20), "queries"), (dict(requests=2**20 + 1), "requests"),
    (dict(width=2**27), "too long"), (dict(ldq=255), "overlap"), (dict(ldo=255), "overlap"), (dict(ldq=2**29), "apart"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(causal=2), "causal"), (dict(causal=0, window=4), "window"),
    (dict(starts=None), "starts"), (dict(lengths=None), "null"), (dict(table=None), "null"), (dict(q=None), "queries"),
    (dict(out=None), "output"), (dict(q=D + 1), "unaligned"), (dict(out=D + 1), "unaligned"), (dict(work_bytes=64), "workspace"), (dict(work=None), "null"),
    (dict(q_type=3), "type"), (dict(out_type=-1), "type"), (dict(work=D + 8), "aligned"),
    (dict(out=D), "overlaps"), (dict(out=D, ldq=768), "overlaps"), (dict(out=D + 6 * 512 - 16), "overlaps"), (dict(q=(1 << 20) + 16, out_type=0), "overlaps"),
])
def test_attention(change, word):
    if B.device_count() < 1 and ("work" in change or "work_bytes" in change):
        word = "device"  # the size of the workspace hangs on its CUs
    refused(B.lib().bsq_kv4_attention(*attention_args(**change)), word)


def test_empty_calls_succeed():
    L = B.lib()
    empty = cache(d_pages=None)
    assert L.bsq_rope(rope(), None, None, 0, 0, 2, 64, 128, 0, None, 128, None) == 0
    assert L.bsq_rope(rope(), None, None, 0, 5, 0, 64, 0, 0, None, 0, None) == 0
    assert L.bsq_kv4_append(empty, None, None, None, 0, 0, None, 0, 0, None, 0, None, 128, None, 128, None) == 0
    assert L.bsq_kv4_read(empty, None, 0, 0, None, 0, None, 0, None) == 0
    assert L.bsq_kv4_read(cache(), None, 4, 0, None, 0, None, 0, None) == 0


class Untouched:
    """In the place of device memory: nothing may be asked of it."""

    def __init__(self, nbytes):
        raise AssertionError("device memory was asked for")

    @staticmethod
    def from_array(a):
        raise AssertionError("an upload was asked for")


def test_binding(monkeypatch):
    monkeypatch.setattr(B, "DeviceBuffer", Untouched)

    def no(call, word):
        with pytest.raises(ValueError, match=word):
            call()

    def zeros(*shape):
        return np.zeros(shape, np.float32)

    no(lambda: B.Turn(zeros(2, 2)), "frequencies")
    no(lambda: B.Kv4Cache(0, 16, 1, 8, 1, 1), "sizes")
    with pytest.raises(B.BsqError, match="page"):
        B.Kv4Cache(4, 15, 1, 8, 1, 1)
    turn = object.__new__(B.Turn)
    turn.dims = 16
    no(lambda: B.rope(zeros(4, 8), np.zeros(4), turn), "tokens x heads")
    no(lambda: B.rope(zeros(4, 2, 16), np.zeros(3), turn), "position")
    no(lambda: B.rope(zeros(4, 2, 8), np.zeros(4), turn), "turning")
    c = object.__new__(B.Kv4Cache)
    c.requests, c.heads, c.dim, c.tokens = 3, 2, 8, None
    no(lambda: c.step(np.zeros(4)), "3 requests")
    no(lambda: c.append(zeros(4, 2, 8), zeros(4, 2, 8)), "step")
    c.tokens = 4
    no(lambda: c.append(zeros(5, 2, 8), zeros(4, 2, 8)), "keys")
    no(lambda: c.append(zeros(4, 2, 8), zeros(4, 1, 8)), "values")
    no(lambda: c.append(zeros(4, 2, 8), zeros(4, 2, 8), zeros(4, 2, 7)), "queries")
    no(lambda: c.append(zeros(4, 2, 8), zeros(4, 2, 8), turn=turn), "turning")
    no(lambda: c.attend(zeros(4, 3, 8)), "multiple")
    no(lambda: c.attend(zeros(4, 16)), "queries")
    no(lambda: c.read(np.zeros((2, 2))), "slots")
