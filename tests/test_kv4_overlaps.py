"""Which results of the paged cache's calls count as lying on what the call reads
(include/bitsqz_llm_c.h, group 7), without a GPU: the check runs before any device
work, and pointers are never reached."""
import pytest

import bitsqz_amd as B
from test_kv4_refusals import D, attention_args, refused, rope

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
