"""The size queries of the MX4 and expert-layer calls (include/bitsqz_llm_c.h,
group 6): what they answer where there is no answer.  Without a GPU."""
import os
import subprocess
import sys

import pytest

import bitsqz_amd as B

NONE = 2**64 - 1  # no size


def answer(query, *args):
    """(size, message) of a query in a process without a device."""
    code = ("import sys; sys.path.insert(0, sys.argv[1]); import bitsqz_amd as B\n"
            "print(getattr(B.lib(), sys.argv[2])(*map(int, sys.argv[3:])), B.lib().bsq_last_error().decode())")
    r = subprocess.run([sys.executable, "-c", code, B.HERE, query, *map(str, args)], capture_output=True, text=True,
                       env=dict(os.environ, HIP_VISIBLE_DEVICES="-1"), timeout=120)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    size, _, message = r.stdout.strip().partition(" ")
    return int(size), message


@pytest.mark.parametrize("query,args", [("bsq_mx4_product_workspace", (64, 4096, 4096)),
                                        ("bsq_mx4_linear_workspace", (100, 256, 256)),
                                        ("bsq_mx4_linear_backward_workspace", (2048, 4096, 4096))])
def test_no_device_is_an_error_of_the_query(query, args):
    # how a product is cut depends on the device: without one there is no size,
    # and the process lives on
    size, message = answer(query, *args)
    assert size == NONE and message


def test_few_rows_need_no_device():
    assert answer("bsq_mx4_product_workspace", 16, 4096, 4096) == (0, "")


@pytest.mark.parametrize("query,args", [
    ("bsq_mx4_product_workspace", (1 << 31, 8, 8)), ("bsq_mx4_product_workspace", (1 << 32, 8, 8)),
    ("bsq_mx4_product_workspace", (8, (1 << 32) + 4, 8)), ("bsq_mx4_product_workspace", (8, 8, (1 << 22) + 1)),
    ("bsq_mx4_linear_workspace", ((1 << 32) + 1, 8, 8)), ("bsq_mx4_linear_workspace", (8, 8, 1 << 40)),
    ("bsq_mx4_linear_backward_workspace", ((1 << 22) + 1, 8, 8)),
    ("bsq_mx4_linear_backward_workspace", (8, (1 << 22) + 1, 8)),
    ("bsq_mx4_linear_backward_workspace", (8, 8, 1 << 33)),
    ("bsq_moe_linear_workspace", (1 << 62, 4, 8, 8, 8)), ("bsq_moe_linear_workspace", (4, 0, 8, 8, 8)),
    ("bsq_moe_linear_workspace", (4, 2, 8, 1 << 60, 8)), ("bsq_moe_linear_workspace", (4, 2, 8, 8, 1025)),
    ("bsq_moe_linear_backward_workspace", (1 << 62, 4, 8, 8, 8)), ("bsq_moe_linear_backward_workspace", (4, 65, 8, 8, 8)),
    ("bsq_moe_linear_backward_workspace", (4, 2, 1 << 40, 8, 8)), ("bsq_moe_linear_backward_workspace", (4, 2, 8, 8, 0)),
])
def test_sizes_that_no_call_takes(query, args):
    L = B.lib()
    assert getattr(L, query)(*args) == NONE
    assert b"mx4: up to" in L.bsq_last_error() or b"moe linear" in L.bsq_last_error()


def test_the_binding_reports_it():
    with pytest.raises(B.BsqError, match="up to 2\\^31 rows"):
        B.workspace("bsq_mx4_product_workspace", 1 << 32, 8, 8)
    assert B.workspace("bsq_moe_linear_workspace", 4, 2, 8, 300, 5) == B.lib().bsq_moe_linear_workspace(4, 2, 8, 300, 5)
