"""Results in other columns of the rows that they are computed from: apart from
them, though their spans cross."""
import numpy as np
import pytest

import bitsqz_amd as B
from test_gpu_mx4 import stored

pytestmark = pytest.mark.gpu

TOKENS, HEADS, DIM = 37, 2, 64
WIDTH = HEADS * DIM


def rows(rng, columns, type=B.TYPE_BF16):
    raw, _ = stored(rng.standard_normal((TOKENS, columns)), type)
    return raw, B.DeviceBuffer.from_array(raw)


def same(buffer, raw, at, apart, width=WIDTH):
    """The columns from `at` hold what `apart` holds, the others what they held."""
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    got = buffer.download(raw.dtype, raw.size).reshape(raw.shape)
    want = raw.copy()
    want[:, at: at + width] = apart.download(raw.dtype, TOKENS * width).reshape(TOKENS, width)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("first", [True, False])  # the result ahead of its input, or behind
def test_rope(first):
    L, (raw, x) = B.lib(), rows(np.random.default_rng(1), 2 * WIDTH + 6)
    turn, p = B.Turn(B.rope_frequencies(DIM)[0]), B.DeviceBuffer.from_array(np.arange(TOKENS, dtype=np.int32))
    source, to = (WIDTH + 6, 0) if first else (0, WIDTH + 6)
    apart = B.DeviceBuffer(2 * TOKENS * WIDTH)
    row = raw.shape[1]
    for out, ld in ((apart.value, WIDTH), (x.value + 2 * to, row)):
        B.check(L.bsq_rope(turn.rope, p.ptr, x.value + 2 * source, 1, TOKENS, HEADS, DIM, row, 0, out, ld, None), "rope")
    same(x, raw, to, apart)


def test_append():
    # queries, keys, values, and room for the turned queries between them
    L, (raw, x) = B.lib(), rows(np.random.default_rng(2), 4 * WIDTH)
    turn, p = B.Turn(B.rope_frequencies(DIM)[0]), B.DeviceBuffer.from_array(np.arange(TOKENS, dtype=np.int32))
    pools = [B.DeviceBuffer(L.bsq_kv4_cache_bytes(3, 16, HEADS, DIM)) for _ in range(2)]
    apart, row = B.DeviceBuffer(2 * TOKENS * WIDTH), raw.shape[1]
    for pool, out, ld in ((pools[0], apart.value, WIDTH), (pools[1], x.value + 4 * WIDTH, row)):
        pool.zero()
        cache = B.Kv4Pages(pool.value, 3, 16, HEADS, DIM)
        B.check(L.bsq_kv4_append(cache, turn.rope, p.ptr, p.ptr, TOKENS, 1, x.value, HEADS, row, out, ld, x.value + 2 * WIDTH,
                                 row, x.value + 6 * WIDTH, row, None), "append")
    same(x, raw, 2 * WIDTH, apart)
    assert np.array_equal(*(pool.download(np.uint8, pool.nbytes) for pool in pools))


@pytest.mark.parametrize("first", [True, False])
def test_attention(first):
    L, (raw, x) = B.lib(), rows(np.random.default_rng(3), 2 * WIDTH)
    c = B.Kv4Cache(4, 16, HEADS, DIM, 1, 4)
    c.step([TOKENS])
    k, v = (np.random.default_rng(i).standard_normal((TOKENS, HEADS, DIM)).astype(np.float32) for i in (4, 5))
    c.append(k, v)
    source, to = (WIDTH, 0) if first else (0, WIDTH)
    apart, row = B.DeviceBuffer(2 * TOKENS * WIDTH), raw.shape[1]
    work = B.DeviceBuffer(B.workspace("bsq_kv4_attention_workspace", c.cache, c.width, 1, TOKENS, TOKENS, HEADS))
    for out, ld in ((apart.value, WIDTH), (x.value + 2 * to, row)):
        B.check(L.bsq_kv4_attention(c.cache, c.table.ptr, c.width, c.lengths.ptr, c.starts.ptr, 1, x.value + 2 * source, 1, TOKENS,
                                    TOKENS, HEADS, row, 0.125, 1, 0, out, 1, ld, None, work.ptr, work.nbytes, None), "attention")
    same(x, raw, to, apart)
