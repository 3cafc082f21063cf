"""Which results of the paged cache's calls count as lying on what the call reads
(include/bitsqz_llm_c.h, group 7), without a GPU: the check runs before any device
work, and pointers are never reached."""
import pytest

import bitsqz_amd as B
from test_kv4_refusals import D, attention_args, cache, refused, rope

Q, K, V = 256, 128, 128  # columns of one product's rows, BF16
ROW = Q + K + V


def append(**change):
    a = dict(cache=cache(), rope=rope(), positions=D, slots=D, tokens=4, type=1, q=D, q_heads=4, ldq=ROW, q_out=D, ldqo=ROW,
             k=D + 2 * Q, ldk=ROW, v=D + 2 * (Q + K), ldv=ROW, stream=None)
    a.update(change)
    return B.lib().bsq_kv4_append(*a.values())


@pytest.mark.parametrize("change", [
    # on the keys, on the values, on the end of either, in rows of the same distance
    dict(q_out=D + 2 * Q), dict(q_out=D + 2 * (Q + K) - 2), dict(q_out=D + 2 * (ROW - 1)),
    # in place, and keys or values among the queries, or in rows of another distance
    dict(k=D), dict(v=D + 2 * Q - 16), dict(ldk=ROW - 8),
    # beside the product's rows
    dict(q_out=1 << 20, ldqo=Q, k=1 << 20, ldk=K), dict(q_out=1 << 20, ldqo=Q, v=(1 << 20) + 2 * 4 * Q - 2, ldv=V),
    dict(q_out=1 << 20, ldqo=Q, k=(1 << 20) - 2, ldk=K),
])
def test_append(change):
    refused(append(**change), "overlaps")


def test_append_of_nothing_to_turn():
    # in place and without positions no query is written
    a = dict(rope=None, k=D, v=D, positions=None)
    if B.device_count() < 1:
        assert append(**a) == 1 and "overlap" not in B.lib().bsq_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(out=D + 2 * 255, ldq=512, ldo=512), dict(q=D + 2 * 255, out=D, ldq=512, ldo=512),  # a column in common
    dict(out=D + 512, ldq=512, ldo=256, out_type=0, q_type=1),  # columns 512 bytes on, rows 1024 bytes apart, FP32 of 1024
    dict(out=D + 512, ldq=512, ldo=513),
])
def test_attention(change):
    refused(B.lib().bsq_kv4_attention(*attention_args(**change)), "overlaps")


@pytest.mark.parametrize("change", [
    dict(out=D + 254, ldx=256, ldo=256), dict(x=D + 254, out=D, ldx=256, ldo=256), dict(out=D + 256, ldx=256, ldo=257),
])
def test_rope(change):
    a = dict(rope=rope(), positions=D, x=D, type=1, tokens=4, heads=2, dim=64, ldx=128, back=0, out=1 << 20, ldo=128, stream=None)
    a.update(change)
    refused(B.lib().bsq_rope(*a.values()), "overlaps")


@pytest.mark.parametrize("change", [
    dict(), dict(v=D + 2 * 127), dict(k=D + 2 * 3 * 128, v=D), dict(v=D + 256, ldk=256, ldv=255), dict(v=D + 254, ldk=256, ldv=256),
])
def test_read(change):
    a = dict(cache=cache(), slots=D, tokens=4, type=1, k=D, ldk=128, v=D, ldv=128, stream=None)
    a.update(change)
    refused(B.lib().bsq_kv4_read(*a.values()), "overlap")
