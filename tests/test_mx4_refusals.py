"""What the MX4 and expert-layer entry points refuse (include/bitsqz_llm_c.h,
group 6), without a GPU: the checks run before any device work.  Pointers that
are never reached are small integers of the right alignment."""
import numpy as np
import pytest

import bitsqz_amd as B

D = 4096  # a pointer that is not followed


def refused(rc, word):
    msg = B.lib().bsq_last_error().decode()
    assert rc == 1 and word in msg, (rc, msg)


def test_packed_sizes():
    L = B.lib()
    for rows, cols in ((0, 5), (1, 1), (3, 256), (3, 257), (1 << 20, 1 << 20)):
        slices = -(-cols // 256)
        assert L.bsq_mx4_codes_bytes(rows, cols) == rows * slices * 128
        assert L.bsq_mx4_scales_bytes(rows, cols) == rows * slices * 8


def test_empty_calls_succeed():
    L = B.lib()
    assert L.bsq_mx4_encode(None, 0, 1, 0, 8, 8, 0, None, None, None, None, None) == 0
    assert L.bsq_mx4_encode(None, 0, 0, 4, 8, 8, 0, None, None, None, None, None) == 0
    assert L.bsq_mx4_decode(None, None, 3, 0, None, 1, 0, None) == 0
    assert L.bsq_mx4_product(None, None, 0, None, None, 5, 7, None, 0, 5, None, 0, None) == 0
    assert L.bsq_mx4_linear(None, 0, 0, 7, 7, None, None, 5, None, 0, 5, None, None, None, 0, None) == 0
    assert L.bsq_moe_route(None, 0, 0, 8, 8, None, 0, 1, 1, 2, 1, 1.0, None, None, None) == 0
    assert L.bsq_moe_combine(None, 0, 0, 2, 8, None, None, 4, None, 0, 8, None) == 0


@pytest.mark.parametrize("args,word", [
    ((D, 3, 1, 4, 8, 8, 0, D, D, None, None, None), "type"),
    ((D, 0, 1, 4, 8, 7, 0, D, D, None, None, None), "overlap"),
    ((None, 0, 1, 4, 8, 8, 0, D, D, None, None, None), "null input"),
    ((D + 2, 0, 1, 4, 8, 8, 0, D, D, None, None, None), "unaligned"),
    ((D + 1, 1, 1, 4, 8, 8, 0, D, D, None, None, None), "unaligned"),
    ((D, 0, 1, 4, 8, 8, 0, None, None, None, None, None), "null output"),
    ((D, 0, 1, 4, 8, 8, 0, D, None, None, None, None), "scales"),
    ((D, 0, 1, 4, 8, 8, 0, D, D, None, D, None), "scales"),
    ((D, 0, 1, 4, 8, 8, 0, D + 8, D, None, None, None), "aligned"),
    ((D, 0, 1, 4, 8, 8, 0, D, D + 4, None, None, None), "aligned"),
    ((D, 0, 1, 1 << 32, 8, 8, 0, D, D, None, None, None), "rows"),
    ((D, 0, 1, 4, (1 << 22) + 1, 1 << 23, 0, D, D, None, None, None), "values a row"),
    ((D, 0, 1, (1 << 22) + 1, 8, 8, 0, None, None, D, D, None), "values a row"),
])
def test_encode(args, word):
    refused(B.lib().bsq_mx4_encode(*args), word)


@pytest.mark.parametrize("args,word", [
    ((D, D, 4, 8, D, 7, 8, None), "type"),
    ((D, D, 4, 8, D, 0, 7, None), "overlap"),
    ((None, D, 4, 8, D, 0, 8, None), "null"),
    ((D, D, 4, 8, None, 0, 8, None), "null"),
    ((D, D, 4, 8, D + 1, 1, 8, None), "unaligned"),
])
def test_decode(args, word):
    refused(B.lib().bsq_mx4_decode(*args), word)


@pytest.mark.parametrize("args,word", [
    ((D, D, 4, D, D, 8, 0, D, 0, 8, None, 0, None), "no values"),
    ((D, D, 4, D, D, 8, 16, D, -1, 8, None, 0, None), "type"),
    ((D, D, 4, D, D, 8, 16, D, 0, 7, None, 0, None), "overlap"),
    ((D, D, 4, None, D, 8, 16, D, 0, 8, None, 0, None), "null"),
    ((D, D, 4, D, D, 8, 16, None, 0, 8, None, 0, None), "null output"),
    ((D, D, 4, D, D, 8, 16, D + 2, 0, 8, None, 0, None), "unaligned"),
    ((D, D, 1 << 31, D, D, 8, 16, D, 0, 8, None, 0, None), "rows"),
])
def test_product(args, word):
    refused(B.lib().bsq_mx4_product(*args), word)


def test_linear():
    L = B.lib()
    need = L.bsq_mx4_linear_workspace(4, 8, 300)
    assert need >= 4 * 2 * 136

    def call(x=D, xt=None, m=4, k=300, ldx=300, w=D, n=8, out=D, ldo=8, tc=None, ts=None, work=D, size=need, t=0):
        return L.bsq_mx4_linear(x, t, m, k, ldx, w, w, n, out, 0, ldo, tc, ts, work, size, None)

    refused(call(t=9), "type")
    refused(call(ldx=299), "overlap")
    refused(call(ldo=7), "overlap")
    refused(call(k=0), "no inputs")
    refused(call(x=None), "null")
    refused(call(x=D + 2), "unaligned")
    refused(call(out=D + 2), "unaligned")
    refused(call(w=None), "null")
    refused(call(w=D + 8), "aligned")
    refused(call(tc=D), "scales")
    refused(call(size=need - 1), "workspace")
    refused(call(work=None), "null")
    refused(call(work=D + 8), "aligned")
    refused(call(m=(1 << 22) + 1, tc=D, ts=D, size=1 << 60), "values a row")


def test_linear_backward():
    L = B.lib()
    need = L.bsq_mx4_linear_backward_workspace(4, 8, 300)

    def call(dy=D, t=0, m=4, n=8, ldy=8, xt=D, wt=D, k=300, dx=D, lddx=300, dw=D, lddw=300, g=0, work=D, size=need):
        return L.bsq_mx4_linear_backward(dy, t, m, n, ldy, xt, xt, wt, wt, k, dx, lddx, dw, lddw, g, work, size, None)

    refused(call(t=-1), "type")
    refused(call(g=3), "type")
    refused(call(m=0), "empty")
    refused(call(ldy=7), "overlap")
    refused(call(lddx=299), "overlap")
    refused(call(lddw=299), "overlap")
    refused(call(dy=None), "null")
    refused(call(xt=None), "null")
    refused(call(wt=None), "null")
    refused(call(size=need - 1), "workspace")
    assert call(dx=None, dw=None) == 0


@pytest.mark.parametrize("change,word", [
    (dict(t=3), "type"), (dict(e=0), "experts"), (dict(e=1025, ld=1025), "experts"), (dict(k=0), "experts a token"),
    (dict(k=9), "experts a token"), (dict(e=100, ld=100, k=65), "experts a token"), (dict(s=2), "scoring"),
    (dict(g=3), "groups"), (dict(g=0), "groups"), (dict(e=128, ld=128, g=128), "groups"), (dict(g=4, kept=5), "kept"),
    (dict(g=4, kept=0), "kept"), (dict(ld=7), "overlap"), (dict(x=None), "null"), (dict(ids=None), "null"),
    (dict(w=None), "null"), (dict(x=D + 2), "unaligned"), (dict(tokens=1 << 31), "tokens"),
])
def test_route(change, word):
    a = dict(x=D, t=0, tokens=3, e=8, ld=8, s=0, g=1, kept=1, k=2, ids=D, w=D) | change
    refused(B.lib().bsq_moe_route(a["x"], a["t"], a["tokens"], a["e"], a["ld"], None, a["s"], a["g"], a["kept"], a["k"], 1,
                                  1.0, a["ids"], a["w"], None), word)


def test_route_backward_plan_combine():
    L = B.lib()
    refused(L.bsq_moe_route_backward(D, 0, 3, 8, 8, 0, 2, 1, 1.0, D, D, D, 7, None), "overlap")
    refused(L.bsq_moe_route_backward(D, 0, 3, 8, 8, 0, 2, 1, 1.0, D, D, None, 8, None), "null")
    refused(L.bsq_moe_route_backward(D, 0, 3, 8, 8, 2, 2, 1, 1.0, D, D, D, 8, None), "scoring")
    refused(L.bsq_moe_plan(D, 10, 0, D, D, None), "experts")
    refused(L.bsq_moe_plan(D, 1 << 31, 4, D, D, None), "pairs")
    refused(L.bsq_moe_plan(None, 10, 4, D, D, None), "null")
    refused(L.bsq_moe_plan(D, 10, 4, None, D, None), "null")
    refused(L.bsq_moe_combine(D, 5, 3, 2, 8, D, D, 4, D, 0, 8, None), "type")
    refused(L.bsq_moe_combine(D, 0, 3, 2, 8, D, D, 4, D, 0, 7, None), "overlap")
    refused(L.bsq_moe_combine(D, 0, 3, 2, 8, None, D, 4, D, 0, 8, None), "null")
    refused(L.bsq_moe_combine(D, 0, 1 << 31, 2, 8, D, D, 4, D, 0, 8, None), "tokens")


def test_layer():
    L = B.lib()
    need = L.bsq_moe_linear_workspace(4, 2, 8, 300, 5)

    def call(x=D, t=0, m=4, inputs=300, ldx=300, ids=D, weights=D, k=2, w=D, e=5, n=8, off=D, order=D, y=D, yt=0, out=D,
             ot=0, ldo=8, work=D, size=need):
        return L.bsq_moe_linear(x, t, m, inputs, ldx, ids, weights, k, w, w, e, n, off, order, y, yt, out, ot, ldo, work,
                                size, None)

    for change, word in ((dict(t=4), "type"), (dict(yt=4), "type"), (dict(ot=-1), "type"), (dict(e=0), "experts"),
                         (dict(k=0), "experts a token"), (dict(k=65), "experts a token"), (dict(n=0), "outputs"),
                         (dict(inputs=0), "inputs"), (dict(ldx=299), "overlap"), (dict(ldo=7), "overlap"),
                         (dict(x=None), "null"), (dict(ids=None), "null"), (dict(off=None), "null"), (dict(y=None), "null"),
                         (dict(w=None), "null"), (dict(w=D + 8), "aligned"), (dict(x=D + 2), "unaligned"),
                         (dict(y=D + 2), "unaligned"), (dict(out=D + 2), "unaligned"), (dict(size=need - 1), "workspace"),
                         (dict(work=D + 8), "aligned"), (dict(m=1 << 31), "tokens")):
        refused(call(**change), word)

    need = L.bsq_moe_linear_backward_workspace(4, 2, 8, 300, 5)

    def back(dy=D, t=0, m=4, n=8, ldd=8, x=D, xt=0, inputs=300, ldx=300, ids=D, weights=D, k=2, off=D, order=D, y=D, yt=0,
             wt=D, e=5, dx=D, lddx=300, dweights=D, dw=D, g=0, work=D, size=need):
        return L.bsq_moe_linear_backward(dy, t, m, n, ldd, x, xt, inputs, ldx, ids, weights, k, off, order, y, yt, wt, wt, e,
                                         dx, lddx, dweights, dw, g, work, size, None)

    for change, word in ((dict(t=4), "type"), (dict(g=4), "type"), (dict(ldd=7), "overlap"), (dict(ldx=299), "overlap"),
                         (dict(lddx=299), "overlap"), (dict(dy=None), "null"), (dict(order=None), "null"),
                         (dict(off=None), "null"), (dict(wt=None), "columns"), (dict(wt=D + 8), "aligned"),
                         (dict(y=None), "needs y"), (dict(x=None), "needs x"), (dict(size=need - 1), "workspace"),
                         (dict(work=D + 8), "aligned"), (dict(dx=D + 2), "unaligned"), (dict(dw=D + 2), "unaligned")):
        refused(back(**change), word)


def test_bf16_conversion_of_the_binding():
    x = np.array([1.0, 1.00390625, 1.01171875, -0.0, 3.4e38, np.inf, -np.inf, 1e-40], np.float32)
    b = B.to_bf16(x)
    assert b.tolist()[:4] == [0x3F80, 0x3F80, 0x3F82, 0x8000] and b[4] == 0x7F80 and b[5] == 0x7F80 and b[6] == 0xFF80
    assert np.isnan(B.from_bf16(B.to_bf16(np.array([np.nan], np.float32)))).all()


def test_the_experts_weight_gradient_takes_so_many_pairs():
    """A row of its operands is 128 bytes a slice of 256 pairs, and 256 of them lie within 32 bits."""
    L = B.lib()

    def back(tokens, dw):
        return L.bsq_moe_linear_backward(D, 0, tokens, 8, 8, D, 0, 300, 300, D, D, 16, D, D, D, 0, D, D, 5, None, 300, None, dw,
                                         0, D, 0, None)

    refused(back(1 << 21, D), "too many pairs")
    refused(back((1 << 21) - 80, D), "workspace")  # within the limit: the next check's turn
    refused(back(1 << 21, None), "workspace")
