"""Scales of attention that FP32 does not hold once they are turned to powers of two,
without a GPU."""
import pytest

import bitsqz_amd as B
from test_kv4_refusals import attention_args, refused


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38])
def test_scales_times_the_logarithm(scale):
    # log2(e) = 1.4427: from 2.3586e38 on the product is past FP32's 3.4028e38
    refused(B.lib().bsq_kv4_attention(*attention_args(scale=scale)), "scale")
