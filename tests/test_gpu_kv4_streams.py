"""Steps over the paged MX4 cache on streams of the caller's, captured and
replayed, beside one another, and from the example."""
import ctypes
import os
import sys

import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B
from test_gpu_mx4 import Hip, stored, values

pytestmark = pytest.mark.gpu

PAGE, HEADS, QUERIES, DIM, REQUESTS, WIDTH = 16, 2, 6, 64, 4, 20


class Step:
    """Buffers of a step of up to `tokens` tokens: plan, append in place, attention."""

    def __init__(self, tokens, most, work=None):
        self.tokens, self.most = tokens, most
        self.row = (QUERIES + 2 * HEADS) * DIM
        pages = REQUESTS * WIDTH
        self.pool = B.DeviceBuffer(B.lib().bsq_kv4_cache_bytes(pages, PAGE, HEADS, DIM))
        self.pool.zero()
        self.cache = B.Kv4Pages(self.pool.value, pages, PAGE, HEADS, DIM)
        self.table = B.DeviceBuffer.from_array(np.full((REQUESTS, WIDTH), -1, np.int32))
        self.free = B.DeviceBuffer.from_array(np.arange(pages, dtype=np.int32))
        self.left = B.DeviceBuffer.from_array(np.array([pages, 0], np.int32))
        self.lengths = B.DeviceBuffer.from_array(np.zeros(REQUESTS, np.int32))
        self.new = B.DeviceBuffer(4 * REQUESTS)
        self.starts, self.positions, self.slots = B.DeviceBuffer(4 * REQUESTS + 4), B.DeviceBuffer(4 * tokens), B.DeviceBuffer(4 * tokens)
        self.x = B.DeviceBuffer(2 * tokens * self.row)
        self.out, self.lse = B.DeviceBuffer(2 * tokens * QUERIES * DIM), B.DeviceBuffer(4 * tokens * QUERIES)
        need = max(B.workspace("bsq_kv4_plan_workspace", REQUESTS),
                   B.workspace("bsq_kv4_attention_workspace", self.cache, WIDTH, REQUESTS, tokens, most, QUERIES))
        self.work = work if work is not None else B.DeviceBuffer(need)
        assert self.work.nbytes >= need
        self.turn = B.Turn(B.rope_frequencies(DIM)[0])

    def inputs(self, rng, new):
        x = stored(rng.standard_normal((self.tokens, self.row)), B.TYPE_BF16)[0]
        self.x.upload(x)
        self.new.upload(np.array(new, np.int32))

    def run(self, stream):
        L, at = B.lib(), self.x.value
        B.check(L.bsq_kv4_plan(self.lengths.ptr, self.new.ptr, REQUESTS, self.table.ptr, WIDTH, PAGE, self.free.ptr,
                               REQUESTS * WIDTH, self.left.ptr, self.lengths.ptr, self.left.ptr, self.starts.ptr, self.tokens,
                               None, self.positions.ptr, self.slots.ptr, self.work.ptr, self.work.nbytes, stream), "plan")
        B.check(L.bsq_kv4_append(self.cache, self.turn.rope, self.positions.ptr, self.slots.ptr, self.tokens, 1, at, QUERIES,
                                 self.row, at, self.row, at + 2 * QUERIES * DIM, self.row, at + 2 * (QUERIES + HEADS) * DIM,
                                 self.row, stream), "append")
        B.check(L.bsq_kv4_attention(self.cache, self.table.ptr, WIDTH, self.lengths.ptr, self.starts.ptr, REQUESTS, at, 1,
                                    self.tokens, self.most, QUERIES, self.row, 0.125, 1, 0, self.out.ptr, 1, QUERIES * DIM,
                                    self.lse.ptr, self.work.ptr, self.work.nbytes, stream), "attention")

    def results(self):
        n = self.tokens * QUERIES
        return [self.out.download(np.uint16, n * DIM), self.lse.download(np.float32, n), self.lengths.download(np.int32, REQUESTS),
                self.slots.download(np.int32, self.tokens), self.pool.download(np.uint8, self.pool.nbytes)]


def clear(step):
    step.out.zero()
    step.lse.zero()


STEPS = [[20, 3, 0, 90], [1, 1, 0, 1], [1, 1, 44, 1], [1, -1, 1, 1], [64, 7, 1, 1], [1, 1, 1, -1], [1, 1, 1, 1]]


def test_captured_steps_of_two_sizes_with_one_workspace():
    # a graph of 160 places (prompts) and one of 64 share a workspace and take turns;
    # an eager twin has the same steps between the replays
    hip, stream, rng = Hip(), ctypes.c_void_p(), np.random.default_rng(1)
    hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
    eager, played = Step(160, 100), Step(160, 100)
    graphs, views = {}, {}
    for name, tokens in (("large", 160), ("small", 64)):
        view = object.__new__(Step)
        view.__dict__.update(played.__dict__)
        view.tokens, view.most = tokens, 100 if tokens > 64 else 44
        graph, run = ctypes.c_void_p(), ctypes.c_void_p()
        hip("hipStreamBeginCapture", stream, 2)
        view.run(stream)
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
        graphs[name], views[name] = (graph, run), view
    for i, new in enumerate(STEPS):
        name = "large" if sum(max(n, 0) for n in new) > 60 or max(new) > 44 else "small"
        seed = int(rng.integers(1 << 30))
        view = views[name]
        full = eager.tokens, eager.most
        eager.tokens, eager.most = view.tokens, view.most
        for step in (eager, view):
            step.inputs(np.random.default_rng(seed), new)
            clear(step)
        eager.run(None)
        B.check(B.lib().bsq_stream_synchronize(None), "sync")
        want = eager.results()
        hip("hipGraphLaunch", graphs[name][1], stream)
        hip("hipStreamSynchronize", stream)
        got = view.results()
        eager.tokens, eager.most = full
        for g, w in zip(got, want):
            assert np.array_equal(g.view(np.uint8), w.view(np.uint8)), (i, name)
    for graph, run in graphs.values():
        hip("hipGraphExecDestroy", run)
        hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", stream)


def test_two_streams_at_once():
    hip, rng = Hip(), np.random.default_rng(2)
    streams = [ctypes.c_void_p() for _ in range(2)]
    for s in streams:
        hip("hipStreamCreateWithFlags", ctypes.byref(s), 1)
    pairs = [(Step(100, 90), Step(100, 90)) for _ in streams]
    for new in ([20, 3, 0, 70], [1, 1, 80, 1], [1, 9, 1, 1]):
        seeds = [int(rng.integers(1 << 30)) for _ in streams]
        for (alone, beside), seed in zip(pairs, seeds):
            for step in (alone, beside):
                step.inputs(np.random.default_rng(seed), new)
                clear(step)
        hip("hipDeviceSynchronize")
        for (_, beside), s in zip(pairs, streams):
            beside.run(s)
        hip("hipDeviceSynchronize")
        for alone, beside in pairs:
            alone.run(None)
            hip("hipDeviceSynchronize")
            for g, w in zip(beside.results(), alone.results()):
                assert np.array_equal(g.view(np.uint8), w.view(np.uint8))
    for s in streams:
        hip("hipStreamDestroy", s)


def test_example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import kv4_generate

    text, off = kv4_generate.generate(6)
    assert [len(t) for t in text] == [11, 37, 26] and all(0 <= v < kv4_generate.VOCABULARY for t in text for v in t)
    assert np.isfinite(off)


def test_a_step_against_the_definition():
    # what the captured steps are compared with, once against 64 bits
    rng = np.random.default_rng(3)
    step = Step(70, 40)
    step.inputs(rng, [33, 0, 2, 30])
    x = values(step.x.download(np.uint16, step.tokens * step.row), 1).reshape(step.tokens, -1, DIM)
    clear(step)
    step.run(None)
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    out, lse, lengths, slots, _ = step.results()
    assert lengths.tolist() == [33, 0, 2, 30] and (slots[65:] == -1).all()
    out = values(out, 1).reshape(step.tokens, QUERIES, DIM)
    q = values(step.x.download(np.uint16, step.tokens * step.row), 1).reshape(step.tokens, -1, DIM)[:, :QUERIES]
    f = B.rope_frequencies(DIM)[0]
    for first, n in ((0, 33), (33, 2), (35, 30)):
        mine = slice(first, first + n)
        host = K.Cache(3, PAGE, HEADS, DIM)
        k = stored(K.turned(x[mine, QUERIES:-HEADS], np.arange(n), f).astype(np.float32), 1)[1]
        for t in range(n):
            host.put(t, k[t], x[first + t, -HEADS:])
        want, _, of = K.attention(host, np.arange(3), n, q[mine], 0.125)
        bound, _, _ = K.attention_bound(of, n, DIM, 1, 0)
        assert (np.abs(out[mine] - want) <= bound + 2.0**-8 * np.abs(want)).all()
    assert (out[65:] == 0).all()
