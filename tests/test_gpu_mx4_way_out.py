"""The way out of the products' tiles (csrc/mx4_gemm.hip): a wave's lanes
exchange 32 rows at a time through LDS, and the next 32 take the same place.
Sums that are exact, rows further apart than their columns, every output type;
tiles of 64 (one block of 32 rows a wave), 128 (two) and 256 (four), with one
team and with several."""
import numpy as np
import pytest

import bitsqz_amd as B
from test_gpu_mx4 import TYPES, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", [(600, 601, 200), (400, 499, 1800), (300, 203, 4000), (2100, 1003, 513), (1024, 1030, 600),
                                   (2300, 2005, 300), (2950, 2947, 256), (5000, 1801, 300)])
def test_rows_and_columns_find_their_places(type, m, n, k):
    rng = np.random.default_rng(m + n)
    x = rng.integers(-2, 3, (m, k)).astype(np.float32)
    w = rng.integers(-2, 3, (n, k)).astype(np.float32)
    x[:, ::32], w[:, ::32] = 4.0, 4.0  # scale 1 in every block
    # one value of a row is its number's, one of a column's its own, in digits
    for i, a in ((1, x), (6, w)):
        for d in range(5):
            a[:, i + d] = (np.arange(len(a)) // 5**d) % 5 - 2
    want = x @ w.T  # below 2^24: exact
    a, b, ld = B.mx4_encode(x), B.mx4_encode(w), n + 5
    t = {B.TYPE_F32: np.float32, B.TYPE_BF16: np.uint16, B.TYPE_F16: np.float16}[type]
    guard = np.full((m, ld), 7, t)
    out = B.DeviceBuffer.from_array(guard)
    work = B.DeviceBuffer(B.workspace("bsq_mx4_product_workspace", m, n, k))
    B.check(B.lib().bsq_mx4_product(a.codes.ptr, a.scales.ptr, m, b.codes.ptr, b.scales.ptr, n, k, out.ptr, type, ld,
                                    work.ptr, work.nbytes, None), "product")
    B.check(B.lib().bsq_stream_synchronize(None), "sync")
    got = out.download(t, m * ld).reshape(m, ld)
    assert np.array_equal(got[:, :n], B.to_bf16(want) if type == B.TYPE_BF16 else want.astype(t))
    assert (got[:, n:] == 7).all()
