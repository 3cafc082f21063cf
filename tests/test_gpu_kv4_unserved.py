"""Requests that a step of the paged MX4 cache did not serve, in the binding."""
import numpy as np
import pytest

import _kv4ref as K
import bitsqz_amd as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_type", [B.TYPE_F32, B.TYPE_BF16])
def test_their_queries_give_zeros(out_type):
    # the second request finds no page; it keeps its keys, and is served later
    rng = np.random.default_rng(1)
    cache = B.Kv4Cache(4, 16, 1, 32, 3, 3)
    turn = B.Turn(B.rope_frequencies(32)[0])

    def rows(n, heads=1):
        return rng.standard_normal((n, heads, 32)).astype(np.float32)

    def step(new):
        places = cache.step(new)
        k, v, q = rows(cache.tokens), rows(cache.tokens), rows(cache.tokens, 2)
        turned = cache.append(k, v, q, turn)
        out, lse = cache.attend(turned, out_type=out_type)
        return places, q, turned, out, lse

    assert step([16, 16, 4])[0]["unserved"] == 0
    before = cache.buffer.download(np.uint8, cache.buffer.nbytes)
    places, q, turned, out, lse = step([0, 17, 2])
    assert places["unserved"] == 1 and places["starts"].tolist() == [0, 0, 17, 19] and (places["slots"][:17] == -1).all()
    assert (out[:17] == 0).all() and (lse[:17] == -np.inf).all()
    assert np.array_equal(turned[:17], q[:17])
    values = B.from_bf16(out) if out_type == B.TYPE_BF16 else out
    assert np.abs(values[17:]).max() > 0 and np.isfinite(lse[17:]).all()
    page = cache.table.download(np.int32, 9).reshape(3, 3)[1, 0]
    after = cache.buffer.download(np.uint8, cache.buffer.nbytes)
    mine = slice(page * 16 * 34, (page + 1) * 16 * 34)
    assert np.array_equal(after[mine], before[mine])
    places, _, _, out, lse = step([0, 3, 1])
    assert places["unserved"] == 0 and np.isfinite(lse).all() and places["lengths"].tolist() == [16, 19, 7]
    assert K.Cache(1, 16, 1, 32).bytes.nbytes == 16 * 34
