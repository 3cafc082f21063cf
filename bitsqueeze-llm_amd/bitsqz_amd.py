"""ctypes binding of the MI355X bitsqz_llm library (lib/libbitsqz_llm_lib.so).

The library is the product: a C-ABI shared library built from csrc/ by
build.py.  This module only binds it for Python callers (the tests and
bench.py): it defines the packed-object structs with the reference's byte
layout (include/bitsqz_llm.hpp:48-93), a small device-buffer helper over the
library's own hipMalloc wrappers, and thin functions named after the
reference's operators.  It never computes anything itself: every function
either calls the library or fails loudly when the library is missing.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libbitsqz_llm_lib.so")

QUANT_NONE, NF4_DQ, NF4 = -1, 10, 11
INPUT_HOST, INPUT_DEVICE = 0, 1
FLAG_SVD, FLAG_OUTLIER, FLAG_ERROR = 1, 2, 4
SECTION_NONE, SECTION_FP32, SECTION_QUANT, SECTION_TOPK = 0, 1, 2, 3


class Section(C.Structure):
    _fields_ = [("offset", C.c_uint64), ("size", C.c_uint64), ("storage", C.c_uint8),
                ("reserved", C.c_uint8 * 7)]


class PackedHeader(C.Structure):
    """bitsqz_llm_array_t (reference include/bitsqz_llm.hpp:55-83), 200 bytes."""
    _fields_ = [
        ("num_rows", C.c_uint16), ("num_columns", C.c_uint16), ("num_elements", C.c_uint32),
        ("outlier_topk_ratio", C.c_float), ("error_correction_topk_ratio", C.c_float),
        ("svd_ranks", C.c_int16), ("svd_niters", C.c_int16), ("effective_rank", C.c_int16),
        ("reserved0", C.c_int16),
        ("svd_uv_format", C.c_int32), ("svd_s_format", C.c_int32),
        ("quantization_only_format", C.c_int32), ("reserved1", C.c_int32),
        ("flags", C.c_uint32),
        ("section_u", Section), ("section_s", Section), ("section_v", Section),
        ("section_direct", Section), ("section_outlier_topk", Section),
        ("section_error_topk", Section),
        ("payload", C.c_void_p),
    ]


assert C.sizeof(PackedHeader) == 200 and PackedHeader.section_u.offset == 48
assert PackedHeader.payload.offset == 192


class Profile(C.Structure):
    """bitsqz_llm_compress_profile_t (reference include/bitsqz_llm.hpp:85-93)."""
    _fields_ = [(n, C.c_double) for n in (
        "topk_separation_latency_ms", "svd_lowrank_cuda_latency_ms",
        "quantization_compress_latency_ms", "reconsturct_quantization_decompress_latency_ms",
        "reconstruct_svd_latency_ms", "error_extraction_latency_ms", "other_latency_ms")]


class DevicePacked(C.Structure):
    """bsq_device_packed_t (include/bitsqz_llm_c.h)."""
    _fields_ = [
        ("header", PackedHeader),
        ("d_flags", C.c_void_p),
        ("d_dense", C.c_void_p * 4), ("d_scales_f32", C.c_void_p * 4),
        ("d_scales_u8", C.c_void_p * 4), ("d_dq_scale", C.c_void_p * 4),
        ("d_codes", C.c_void_p * 4), ("count", C.c_uint64 * 4),
        ("d_topk_idx", C.c_void_p * 2), ("d_topk_val", C.c_void_p * 2),
        ("topk_k", C.c_uint16 * 2),
    ]


_lib = None
P = C.c_void_p


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} missing: run `python bitsqueeze-llm_amd/build.py`")
    L = C.CDLL(LIB_PATH)
    u16, u32, u64, f32, i32 = C.c_uint16, C.c_uint32, C.c_uint64, C.c_float, C.c_int
    sig = {
        "bsq_last_error": (C.c_char_p, []),
        "bsq_version": (C.c_char_p, []),
        "bsq_compress_initialize": (i32, [u16, u16, f32, f32, i32, i32, i32, i32, i32, i32]),
        "bsq_compress_release": (None, []),
        "bsq_decompress_initialize": (i32, [u16, u16, f32, f32, i32, i32, i32, i32]),
        "bsq_decompress_release": (None, []),
        "bsq_compress": (i32, [P, C.POINTER(C.POINTER(PackedHeader)), C.POINTER(Profile)]),
        "bsq_decompress": (i32, [P, P, u32]),
        "bsq_get_packed_size": (u64, [P]),
        "bsq_load_from_buffer": (C.POINTER(PackedHeader), [P, u64]),
        "bsq_free": (None, [P]),
        "bsq_compress_set_sketch": (i32, [P]),
        "bsq_device_compress": (i32, [P, C.POINTER(DevicePacked)]),
        "bsq_device_decompress": (i32, [C.POINTER(DevicePacked), P, u32]),
        "bsq_device_synchronize": (i32, []),
        "bsq_runtime_stream": (P, []),
        "bsq_lanes_initialize": (i32, [i32, u16, u16, f32, f32, i32, i32, i32, i32, i32]),
        "bsq_lanes_roundtrip": (i32, [i32, P, P]),
        "bsq_lanes_stream": (P, [i32]),
        "bsq_lanes_synchronize": (i32, []),
        "bsq_lanes_release": (None, []),
        "bsq_topk_num_columns": (i32, [u16, f32, C.POINTER(u16)]),
        "bsq_topk_select": (i32, [P, u16, u16, u16, P, P, P, P]),
        "bsq_topk_scatter": (i32, [P, P, u16, u16, u16, P, i32, P]),
        "bsq_quant_compress": (i32, [P, u64, i32, P, P, P, P, P]),
        "bsq_quant_decompress": (i32, [u64, i32, P, P, P, P, P, P]),
        "bsq_quant_nf4_codes": (i32, [P, u64, P, P]),
        "bsq_quant_e4m3_encode": (i32, [P, u64, P, P]),
        "bsq_quant_e4m3_decode": (i32, [P, u64, P, P]),
        "bsq_quant_nf4_code_sweep": (i32, [u64, u64, P, P, P]),
        "bsq_nf4_thresholds": (None, [P]),
        "bsq_svd_lowrank": (i32, [P, i32, i32, i32, i32, P, u64, P, P, P, P]),
        "bsq_svd_lowrank_noalloc": (i32, [P, i32, i32, i32, i32, P, u64, P, P, P, P]),
        "bsq_reconstruct_lowrank": (i32, [P, P, P, i32, i32, i32, P, P]),
        "bsq_gaussian_fill": (i32, [P, u64, u64, P]),
        "bsq_device_count": (i32, [C.POINTER(i32)]),
        "bsq_device_malloc": (i32, [C.POINTER(P), u64]),
        "bsq_device_free": (i32, [P]),
        "bsq_memcpy_h2d": (i32, [P, P, u64]),
        "bsq_memcpy_d2h": (i32, [P, P, u64]),
        "bsq_memcpy_d2d": (i32, [P, P, u64]),
        "bsq_device_memset": (i32, [P, i32, u64]),
        "bsq_host_malloc": (i32, [C.POINTER(P), u64]),
        "bsq_host_free": (i32, [P]),
        "bsq_memcpy_h2d_async": (i32, [P, P, u64, P]),
        "bsq_stream_synchronize": (i32, [P]),
        "bsq_event_create": (i32, [C.POINTER(P)]),
        "bsq_event_destroy": (i32, [P]),
        "bsq_event_record": (i32, [P, P]),
        "bsq_event_elapsed_ms": (i32, [P, P, C.POINTER(f32)]),
        "bsq_kernel_timer_start": (i32, []),
        "bsq_copy_kernel": (i32, [P, P, u64, P]),
        "bsq_kernel_timer_stop": (i32, [C.POINTER(C.c_double), C.POINTER(i32)]),
        "bsq_kernel_timer_read": (i32, [i32, C.POINTER(C.c_double), C.POINTER(i32)]),
        "bsq_legacy_compress": (i32, [i32, P, u64, C.POINTER(P)]),
        "bsq_legacy_decompress": (i32, [P, P, u64]),
        "bsq_legacy_packed_size": (C.c_longlong, [P]),
        "bsq_legacy_load": (P, [P, C.c_longlong]),
        "bsq_legacy_free": (None, [P]),
        "bsq_legacy_payload_bytes": (C.c_longlong, [i32, u64]),
        "bsq_legacy_encode_device": (i32, [i32, P, u64, P, P]),
        "bsq_legacy_decode_device": (i32, [i32, P, u64, P, P]),
        "bsq_legacy_sweep": (i32, [i32, u64, u64, P, P]),
        "bsq_mx4_codes_bytes": (u64, [u64, u64]),
        "bsq_mx4_scales_bytes": (u64, [u64, u64]),
        "bsq_mx4_encode": (i32, [P, i32, u64, u64, u64, u64, u64, P, P, P, P, P]),
        "bsq_mx4_decode": (i32, [P, P, u64, u64, P, i32, u64, P]),
        "bsq_mx4_product_workspace": (u64, [u64, u64, u64]),
        "bsq_mx4_product": (i32, [P, P, u64, P, P, u64, u64, P, i32, u64, P, u64, P]),
        "bsq_mx4_linear_workspace": (u64, [u64, u64, u64]),
        "bsq_mx4_linear": (i32, [P, i32, u64, u64, u64, P, P, u64, P, i32, u64, P, P, P, u64, P]),
        "bsq_mx4_linear_backward_workspace": (u64, [u64, u64, u64]),
        "bsq_mx4_linear_backward": (i32, [P, i32, u64, u64, u64, P, P, P, P, u64, P, u64, P, u64, i32, P, u64, P]),
        "bsq_moe_route": (i32, [P, i32, u64, u32, u64, P, i32, u32, u32, u32, i32, f32, P, P, P]),
        "bsq_moe_route_backward": (i32, [P, i32, u64, u32, u64, i32, u32, i32, f32, P, P, P, u64, P]),
        "bsq_moe_plan": (i32, [P, u64, u32, P, P, P]),
        "bsq_moe_combine": (i32, [P, i32, u64, u32, u64, P, P, u32, P, i32, u64, P]),
        "bsq_moe_linear_workspace": (u64, [u64, u32, u64, u64, u32]),
        "bsq_moe_linear": (i32, [P, i32, u64, u64, u64, P, P, u32, P, P, u32, u64, P, P, P, i32, P, i32, u64, P, u64, P]),
        "bsq_moe_linear_backward_workspace": (u64, [u64, u32, u64, u64, u32]),
        "bsq_moe_linear_backward": (i32, [P, i32, u64, u64, u64, P, i32, u64, u64, P, P, u32, P, P, P, i32, P, P, u32, P,
                                          u64, P, P, i32, P, u64, P]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


class BsqError(RuntimeError):
    pass


def check(rc: int, what: str):
    if rc != 0:
        raise BsqError(f"{what} failed: {lib().bsq_last_error().decode()}")


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


# ---------------------------------------------------------------------------
# device memory
# ---------------------------------------------------------------------------
class DeviceBuffer:
    """A hipMalloc'd buffer owned by Python."""

    def __init__(self, nbytes: int):
        self.nbytes = int(nbytes)
        self.ptr = C.c_void_p()
        if self.nbytes:
            check(lib().bsq_device_malloc(C.byref(self.ptr), self.nbytes), "hipMalloc")

    @classmethod
    def from_array(cls, a: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(a)
        b = cls(a.nbytes)
        b.upload(a)
        return b

    def upload(self, a: np.ndarray):
        a = np.ascontiguousarray(a)
        assert a.nbytes <= self.nbytes
        if a.nbytes:
            check(lib().bsq_memcpy_h2d(self.ptr, _ptr(a), a.nbytes), "H2D")

    def download(self, dtype, count: int) -> np.ndarray:
        out = np.empty(count, dtype)
        if out.nbytes:
            assert out.nbytes <= self.nbytes
            check(lib().bsq_memcpy_d2h(_ptr(out), self.ptr, out.nbytes), "D2H")
        return out

    def zero(self):
        if self.nbytes:
            check(lib().bsq_device_memset(self.ptr, 0, self.nbytes), "memset")

    @property
    def value(self):
        return self.ptr.value

    def free(self):
        if self.ptr and self.ptr.value:
            lib().bsq_device_free(self.ptr)
        self.ptr = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class PinnedBuffer:
    """hipHostMalloc'd (page-locked) host memory owned by Python, viewed as a
    flat numpy array of `dtype`."""

    def __init__(self, count: int, dtype=np.float32):
        self.dtype = np.dtype(dtype)
        self.nbytes = int(count) * self.dtype.itemsize
        self.ptr = C.c_void_p()
        check(lib().bsq_host_malloc(C.byref(self.ptr), max(self.nbytes, 1)), "hipHostMalloc")
        buf = (C.c_char * max(self.nbytes, 1)).from_address(self.ptr.value)
        self.array = np.frombuffer(buf, dtype=self.dtype, count=int(count))

    def copy_to_device_async(self, dst: DeviceBuffer, stream=None):
        check(lib().bsq_memcpy_h2d_async(dst.ptr, self.ptr, self.nbytes, stream), "H2D async")

    def free(self):
        if self.ptr and self.ptr.value:
            self.array = None
            lib().bsq_host_free(self.ptr)
        self.ptr = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


TIMER_RECONSTRUCT, TIMER_RANGE_FINDER = 0, 1
TIMER_TOPK_OUTLIER, TIMER_TOPK_ERROR, TIMER_DIRECT_ENCODE, TIMER_DIRECT_DECODE = 2, 3, 4, 5


def kernel_timer_start() -> None:
    """Bracket the timed launch classes of the pipelines (TIMER_*) with HIP events."""
    check(lib().bsq_kernel_timer_start(), "kernel timer start")


def kernel_timer_stop() -> tuple[float, int]:
    """Stop bracketing; returns (summed ms, launches) of the reconstruction GEMMs since the start."""
    ms, n = C.c_double(), C.c_int()
    check(lib().bsq_kernel_timer_stop(C.byref(ms), C.byref(n)), "kernel timer stop")
    return ms.value, n.value


def kernel_timer_read(timer_class: int) -> tuple[float, int]:
    """After kernel_timer_stop: (summed ms, launches) of one class (TIMER_*)."""
    ms, n = C.c_double(), C.c_int()
    check(lib().bsq_kernel_timer_read(timer_class, C.byref(ms), C.byref(n)), "kernel timer read")
    return ms.value, n.value


def device_count() -> int:
    n = C.c_int(0)
    rc = lib().bsq_device_count(C.byref(n))
    return n.value if rc == 0 else 0


class Event:
    def __init__(self):
        self.h = C.c_void_p()
        check(lib().bsq_event_create(C.byref(self.h)), "event create")

    def record(self, stream=None):
        check(lib().bsq_event_record(self.h, stream), "event record")

    def elapsed_ms(self, stop: "Event") -> float:
        ms = C.c_float()
        check(lib().bsq_event_elapsed_ms(self.h, stop.h, C.byref(ms)), "event elapsed")
        return ms.value

    def __del__(self):
        try:
            lib().bsq_event_destroy(self.h)
        except Exception:
            pass


# ---------------------------------------------------------------------------
# public ABI (bitsqz_llm.hpp) through the extern "C" twins
# ---------------------------------------------------------------------------
def compress_initialize(rows, cols, outlier_ratio=0.0, error_ratio=0.0, svd_ranks=-1, svd_niters=2,
                        uv_format=QUANT_NONE, s_format=QUANT_NONE, direct_format=QUANT_NONE,
                        input_location=INPUT_DEVICE) -> int:
    return lib().bsq_compress_initialize(rows, cols, outlier_ratio, error_ratio, svd_ranks, svd_niters,
                                         uv_format, s_format, direct_format, input_location)


def decompress_initialize(rows, cols, outlier_ratio=0.0, error_ratio=0.0, svd_ranks=-1,
                          uv_format=QUANT_NONE, s_format=QUANT_NONE, direct_format=QUANT_NONE) -> int:
    return lib().bsq_decompress_initialize(rows, cols, outlier_ratio, error_ratio, svd_ranks, uv_format,
                                           s_format, direct_format)


def compress_release():
    lib().bsq_compress_release()


def decompress_release():
    lib().bsq_decompress_release()


def packed_bytes(ptr) -> bytes:
    """Bytes of a library-owned packed object (header + payload)."""
    vp = C.cast(ptr, C.c_void_p)
    n = lib().bsq_get_packed_size(vp)
    return C.string_at(vp, n)


def compress(src, profile: bool = False):
    """bitsqz_llm_compress: `src` is a host float32 array (HOST runtime) or a
    DeviceBuffer (DEVICE runtime).  Returns the packed bytes (and profile)."""
    out = C.POINTER(PackedHeader)()
    prof = Profile() if profile else None  # no struct: the two-argument form
    if isinstance(src, DeviceBuffer):
        p = src.ptr
    else:
        src = np.ascontiguousarray(src, np.float32)
        p = _ptr(src)
    check(lib().bsq_compress(p, C.byref(out), C.byref(prof) if profile else None), "bitsqz_llm_compress")
    try:
        data = packed_bytes(out)
    finally:
        lib().bsq_free(C.cast(out, C.c_void_p))
    return (data, prof) if profile else data


def load(buf: bytes):
    """load_bitsqz_llm_from_buffer -> owned pointer (free with free_packed) or None."""
    b = C.create_string_buffer(bytes(buf), len(buf))
    p = lib().bsq_load_from_buffer(b, len(buf))
    return p if p else None


def free_packed(p):
    lib().bsq_free(C.cast(p, C.c_void_p))


def decompress_to_device(buf: bytes, dst: DeviceBuffer, dst_num_elements: int) -> int:
    """bitsqz_llm_decompress of host bytes into `dst`; returns the ABI status."""
    p = load(buf)
    if p is None:
        return 1
    vp = C.cast(p, C.c_void_p)
    try:
        return lib().bsq_decompress(vp, dst.ptr, dst_num_elements)
    finally:
        lib().bsq_free(vp)


def decompress(buf: bytes, rows: int, cols: int) -> np.ndarray:
    dst = DeviceBuffer(rows * cols * 4)
    check(decompress_to_device(buf, dst, rows * cols), "bitsqz_llm_decompress")
    return dst.download(np.float32, rows * cols).reshape(rows, cols)


def topk_num_columns(cols: int, ratio: float) -> int:
    k = C.c_uint16()
    check(lib().bsq_topk_num_columns(cols, ratio, C.byref(k)), "topk_num_columns")
    return k.value


# ---------------------------------------------------------------------------
# module operators
# ---------------------------------------------------------------------------
def topk_select(x: np.ndarray, k: int, separate: bool = False):
    """Per-row top-k: returns (indices u16 rows x k, values f32 rows x k[, residual])."""
    x = np.ascontiguousarray(x, np.float32)
    rows, cols = x.shape
    dx = DeviceBuffer.from_array(x)
    di = DeviceBuffer(max(1, rows * k * 2))
    dv = DeviceBuffer(max(1, rows * k * 4))
    dr = DeviceBuffer(x.nbytes) if separate else None
    check(lib().bsq_topk_select(dx.ptr, rows, cols, k, di.ptr, dv.ptr, dr.ptr if dr else None, None),
          "topk_select")
    check(lib().bsq_stream_synchronize(None), "sync")
    idx = di.download(np.uint16, rows * k).reshape(rows, k)
    val = dv.download(np.float32, rows * k).reshape(rows, k)
    if separate:
        return idx, val, dr.download(np.float32, rows * cols).reshape(rows, cols)
    return idx, val


def topk_scatter(idx: np.ndarray, val: np.ndarray, dense: np.ndarray, accumulate: bool = True) -> np.ndarray:
    dense = np.ascontiguousarray(dense, np.float32)
    rows, cols = dense.shape
    k = idx.shape[1]
    dd = DeviceBuffer.from_array(dense)
    di = DeviceBuffer.from_array(np.ascontiguousarray(idx, np.uint16))
    dv = DeviceBuffer.from_array(np.ascontiguousarray(val, np.float32))
    check(lib().bsq_topk_scatter(di.ptr, dv.ptr, rows, cols, k, dd.ptr, int(accumulate), None), "topk_scatter")
    check(lib().bsq_stream_synchronize(None), "sync")
    return dd.download(np.float32, rows * cols).reshape(rows, cols)


def quant_compress(x: np.ndarray, method: int):
    """Returns (scales, codes, dq): scales f32 (NF4) or u8 (NF4_DQ)."""
    x = np.ascontiguousarray(x, np.float32).ravel()
    n = x.size
    nb, nc = (n + 63) // 64, (n + 1) // 2
    dx = DeviceBuffer.from_array(x)
    dsf = DeviceBuffer(nb * 4)
    dsu = DeviceBuffer(nb)
    ddq = DeviceBuffer(4)
    dc = DeviceBuffer(nc)
    check(lib().bsq_quant_compress(dx.ptr, n, method, dsf.ptr, dsu.ptr, ddq.ptr, dc.ptr, None), "quant_compress")
    check(lib().bsq_stream_synchronize(None), "sync")
    codes = dc.download(np.uint8, nc)
    if method == NF4:
        return dsf.download(np.float32, nb), codes, 0.0
    return dsu.download(np.uint8, nb), codes, float(ddq.download(np.float32, 1)[0])


def quant_decompress(n: int, method: int, scales: np.ndarray, codes: np.ndarray, dq: float = 0.0) -> np.ndarray:
    nb = (n + 63) // 64
    dsf = DeviceBuffer.from_array(np.ascontiguousarray(scales, np.float32)) if method == NF4 else DeviceBuffer(4)
    dsu = DeviceBuffer.from_array(np.ascontiguousarray(scales, np.uint8)) if method == NF4_DQ else DeviceBuffer(4)
    ddq = DeviceBuffer.from_array(np.array([dq], np.float32))
    dc = DeviceBuffer.from_array(np.ascontiguousarray(codes, np.uint8))
    out = DeviceBuffer(n * 4)
    assert scales.size == nb
    check(lib().bsq_quant_decompress(n, method, dsf.ptr, dsu.ptr, ddq.ptr, dc.ptr, out.ptr, None), "quant_decompress")
    check(lib().bsq_stream_synchronize(None), "sync")
    return out.download(np.float32, n)


def _batch(fn_name, src: np.ndarray, out_dtype):
    dsrc = DeviceBuffer.from_array(src)
    dout = DeviceBuffer(max(1, src.size * np.dtype(out_dtype).itemsize))
    check(getattr(lib(), fn_name)(dsrc.ptr, src.size, dout.ptr, None), fn_name)
    check(lib().bsq_stream_synchronize(None), "sync")
    return dout.download(out_dtype, src.size)


def nf4_codes(v: np.ndarray) -> np.ndarray:
    return _batch("bsq_quant_nf4_codes", np.ascontiguousarray(v, np.float32).ravel(), np.uint8)


def e4m3_encode(v: np.ndarray) -> np.ndarray:
    return _batch("bsq_quant_e4m3_encode", np.ascontiguousarray(v, np.float32).ravel(), np.uint8)


def e4m3_decode(c: np.ndarray) -> np.ndarray:
    return _batch("bsq_quant_e4m3_decode", np.ascontiguousarray(c, np.uint8).ravel(), np.float32)


def nf4_code_sweep(lo: int, hi: int):
    dh = DeviceBuffer(16 * 8)
    dc = DeviceBuffer(8)
    check(lib().bsq_quant_nf4_code_sweep(lo, hi, dh.ptr, dc.ptr, None), "nf4 sweep")
    check(lib().bsq_stream_synchronize(None), "sync")
    return dh.download(np.uint64, 16), int(dc.download(np.uint64, 1)[0])


def nf4_thresholds() -> np.ndarray:
    out = np.zeros(15, np.float32)
    lib().bsq_nf4_thresholds(_ptr(out))
    return out


def svd_lowrank(A: np.ndarray, q: int, niter: int, sketch: np.ndarray | None = None, seed: int = 1241):
    A = np.ascontiguousarray(A, np.float32)
    m, n = A.shape
    k = max(1, min(q, m, n))
    dA = DeviceBuffer.from_array(A)
    dR = DeviceBuffer.from_array(np.ascontiguousarray(sketch, np.float32)) if sketch is not None else None
    dU, dS, dV = DeviceBuffer(m * k * 4), DeviceBuffer(k * 4), DeviceBuffer(n * k * 4)
    check(lib().bsq_svd_lowrank(dA.ptr, m, n, q, niter, dR.ptr if dR else None, seed, dU.ptr, dS.ptr, dV.ptr,
                                None), "svd_lowrank")
    return (dU.download(np.float32, m * k).reshape(m, k), dS.download(np.float32, k),
            dV.download(np.float32, n * k).reshape(n, k))


def reconstruct(U: np.ndarray, S: np.ndarray, V: np.ndarray) -> np.ndarray:
    U = np.ascontiguousarray(U, np.float32)
    V = np.ascontiguousarray(V, np.float32)
    m, k = U.shape
    n = V.shape[0]
    dU, dS, dV = DeviceBuffer.from_array(U), DeviceBuffer.from_array(np.ascontiguousarray(S, np.float32)), \
        DeviceBuffer.from_array(V)
    out = DeviceBuffer(m * n * 4)
    check(lib().bsq_reconstruct_lowrank(dU.ptr, dS.ptr, dV.ptr, m, n, k, out.ptr, None), "reconstruct")
    check(lib().bsq_stream_synchronize(None), "sync")
    return out.download(np.float32, m * n).reshape(m, n)


def gaussian(n: int, seed: int) -> np.ndarray:
    d = DeviceBuffer(n * 4)
    check(lib().bsq_gaussian_fill(d.ptr, n, seed, None), "gaussian_fill")
    check(lib().bsq_stream_synchronize(None), "sync")
    return d.download(np.float32, n)


# ---------------------------------------------------------------------------
# device-resident pipeline
# ---------------------------------------------------------------------------
def device_compress(src: DeviceBuffer) -> DevicePacked:
    out = DevicePacked()
    check(lib().bsq_device_compress(src.ptr, C.byref(out)), "bsq_device_compress")
    return out


def device_decompress(packed: DevicePacked, dst: DeviceBuffer, n: int):
    check(lib().bsq_device_decompress(C.byref(packed), dst.ptr, n), "bsq_device_decompress")


def device_synchronize():
    check(lib().bsq_device_synchronize(), "bsq_device_synchronize")


def runtime_stream():
    return lib().bsq_runtime_stream()


# ---------------------------------------------------------------------------
# legacy quantisation formats (include/quantization.hpp)
# ---------------------------------------------------------------------------
LEGACY_Q8_0, LEGACY_Q4_0, LEGACY_Q2_K, LEGACY_BF16, LEGACY_FP16, LEGACY_FP8, LEGACY_FP4 = 0, 1, 2, 3, 4, 5, 6
LEGACY_MXFP8, LEGACY_MXFP4, LEGACY_NVFP4, LEGACY_NF4_DQ, LEGACY_NF4, LEGACY_Q2_K_FAST = 7, 8, 9, 10, 11, 12


def legacy_compress_handle(method: int, x: np.ndarray):
    """quantization_compress of host floats; returns (rc, buffer pointer)."""
    x = np.ascontiguousarray(x, np.float32).ravel()
    out = C.c_void_p()
    rc = lib().bsq_legacy_compress(method, _ptr(x) if x.size else None, x.size, C.byref(out))
    return rc, out


def legacy_compress(method: int, x: np.ndarray) -> bytes:
    """The serialised buffer (quantization_get_packed_size bytes)."""
    rc, h = legacy_compress_handle(method, x)
    check(rc, "quantization_compress")
    try:
        size = lib().bsq_legacy_packed_size(h)
        assert size > 0
        return C.string_at(h, size)
    finally:
        lib().bsq_legacy_free(h)


def legacy_decompress(buf: bytes, n: int, dst_n: int | None = None):
    """load_quantization_from_buffer + quantization_decompress; returns
    (rc, floats) with rc = -1 when the load is refused."""
    raw = C.create_string_buffer(buf, len(buf))
    h = lib().bsq_legacy_load(raw, len(buf))
    if not h:
        return -1, None
    try:
        out = np.zeros(max(n, 1), np.float32)
        rc = lib().bsq_legacy_decompress(h, _ptr(out), n if dst_n is None else dst_n)
        return rc, out[:n]
    finally:
        lib().bsq_legacy_free(h)


def legacy_payload_bytes(method: int, n: int) -> int:
    return int(lib().bsq_legacy_payload_bytes(method, n))


def legacy_encode_device(method: int, x: np.ndarray) -> bytes:
    """Payload image written by the device encoder (pointer fields as the
    device left them)."""
    x = np.ascontiguousarray(x, np.float32).ravel()
    size = legacy_payload_bytes(method, x.size)
    src = DeviceBuffer.from_array(x)
    img = DeviceBuffer(size)
    check(lib().bsq_legacy_encode_device(method, src.ptr, x.size, img.ptr, None), "legacy encode")
    check(lib().bsq_stream_synchronize(None), "sync")
    return img.download(np.uint8, size).tobytes()


def legacy_decode_device(method: int, payload: bytes, n: int) -> np.ndarray:
    img = DeviceBuffer.from_array(np.frombuffer(payload, np.uint8))
    dst = DeviceBuffer(4 * n)
    check(lib().bsq_legacy_decode_device(method, img.ptr, n, dst.ptr, None), "legacy decode")
    check(lib().bsq_stream_synchronize(None), "sync")
    return dst.download(np.float32, n)


def legacy_sweep(kind: int, lo: int, hi: int) -> int:
    d = DeviceBuffer(8)
    d.zero()
    check(lib().bsq_legacy_sweep(kind, lo, hi, d.ptr, None), "legacy sweep")
    check(lib().bsq_stream_synchronize(None), "sync")
    return int(d.download(np.uint64, 1)[0])


# ---------------------------------------------------------------------------
# microscaled 4-bit matrices and the layers that compute with them
# (include/bitsqz_llm_c.h, group 6)
# ---------------------------------------------------------------------------
TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
SCORE_SOFTMAX, SCORE_SIGMOID = 0, 1
_TYPE_NUMPY = {TYPE_F32: np.dtype(np.float32), TYPE_BF16: np.dtype(np.uint16), TYPE_F16: np.dtype(np.float16)}


def to_bf16(x: np.ndarray) -> np.ndarray:
    """Bit patterns (uint16) of the nearest BF16 values, ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u + (0x7FFF + ((u >> 16) & 1)).astype(np.uint32)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), ((u >> 16) | 0x40).astype(np.uint16), r)


def from_bf16(bits: np.ndarray) -> np.ndarray:
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _typed(x: np.ndarray, type: int) -> np.ndarray:
    """Host values in a type's storage (BF16: bit patterns, or floats to round)."""
    x = np.asarray(x)
    if type == TYPE_BF16 and x.dtype != np.uint16:
        return to_bf16(x)
    return np.ascontiguousarray(x, _TYPE_NUMPY[type])


def _agree(ok: bool, what: str):
    """The calls see only pointers: sizes that do not agree are refused here,
    before anything is uploaded."""
    if not ok:
        raise ValueError(what)


def workspace(query: str, *sizes: int) -> int:
    """The bytes that a bsq_*_workspace query gives; raises where there is no size."""
    n = getattr(lib(), query)(*sizes)
    if n == 2**64 - 1:
        raise BsqError(f"{query} failed: {lib().bsq_last_error().decode()}")
    return n


class Mx4:
    """A packed matrix of rows x cols (or several, one after another) on the GPU."""

    def __init__(self, rows: int, cols: int, batch: int = 1):
        self.rows, self.cols, self.batch = rows, cols, batch
        self.codes = DeviceBuffer(batch * lib().bsq_mx4_codes_bytes(rows, cols))
        self.scales = DeviceBuffer(batch * lib().bsq_mx4_scales_bytes(rows, cols))

    def download(self):
        """(codes, scales) as stored: batch * rows x padded cols / 2 and / 32."""
        n = self.batch * self.rows
        return (self.codes.download(np.uint8, self.codes.nbytes).reshape(n, -1),
                self.scales.download(np.uint8, self.scales.nbytes).reshape(n, -1))

    def decode(self, type: int = TYPE_F32) -> np.ndarray:
        n = self.batch * self.rows
        out = DeviceBuffer(n * self.cols * _TYPE_NUMPY[type].itemsize)
        check(lib().bsq_mx4_decode(self.codes.ptr, self.scales.ptr, n, self.cols, out.ptr, type, self.cols, None),
              "mx4_decode")
        check(lib().bsq_stream_synchronize(None), "sync")
        return out.download(_TYPE_NUMPY[type], n * self.cols).reshape(n, self.cols)


def mx4_encode(x: np.ndarray, type: int = TYPE_F32, rows: bool = True, columns: bool = False):
    """The packed rows and / or columns of x (rows x cols, or a batch of those)."""
    x = _typed(x, type)
    _agree(x.ndim in (2, 3), "mx4_encode: x is rows x cols or a batch of those")
    batch, r, c = (1, *x.shape) if x.ndim == 2 else x.shape
    by_row = Mx4(r, c, batch) if rows else None
    by_col = Mx4(c, r, batch) if columns else None
    d = DeviceBuffer.from_array(x)
    check(lib().bsq_mx4_encode(d.ptr, type, batch, r, c, c, r * c, by_row.codes.ptr if rows else None,
                               by_row.scales.ptr if rows else None, by_col.codes.ptr if columns else None,
                               by_col.scales.ptr if columns else None, None), "mx4_encode")
    check(lib().bsq_stream_synchronize(None), "sync")
    return (by_row, by_col) if rows and columns else by_row or by_col


def mx4_product(a: Mx4, b: Mx4, type: int = TYPE_F32) -> np.ndarray:
    _agree(a.batch == b.batch == 1, "mx4_product: a batch of matrices")
    _agree(a.cols == b.cols, f"mx4_product: {a.cols} and {b.cols} columns")
    out = DeviceBuffer(a.rows * b.rows * _TYPE_NUMPY[type].itemsize)
    work = DeviceBuffer(workspace("bsq_mx4_product_workspace", a.rows, b.rows, a.cols))
    check(lib().bsq_mx4_product(a.codes.ptr, a.scales.ptr, a.rows, b.codes.ptr, b.scales.ptr, b.rows, a.cols, out.ptr,
                                type, b.rows, work.ptr, work.nbytes, None), "mx4_product")
    check(lib().bsq_stream_synchronize(None), "sync")
    return out.download(_TYPE_NUMPY[type], a.rows * b.rows).reshape(a.rows, b.rows)


def mx4_linear(x: np.ndarray, w: Mx4, type: int = TYPE_F32, out_type: int = TYPE_F32, keep: bool = False):
    """out = q(x) W^T; with `keep` also the packed transpose of x."""
    x = _typed(x, type)
    _agree(x.ndim == 2, "mx4_linear: x is a matrix")
    _agree(w.batch == 1, "mx4_linear: a batch of weights")
    _agree(x.shape[1] == w.cols, f"mx4_linear: x has {x.shape[1]} columns, the weights {w.cols}")
    m, k = x.shape
    d, out = DeviceBuffer.from_array(x), DeviceBuffer(m * w.rows * _TYPE_NUMPY[out_type].itemsize)
    work = DeviceBuffer(workspace("bsq_mx4_linear_workspace", m, w.rows, k))
    xt = Mx4(k, m) if keep else None
    check(lib().bsq_mx4_linear(d.ptr, type, m, k, k, w.codes.ptr, w.scales.ptr, w.rows, out.ptr, out_type, w.rows,
                               xt.codes.ptr if keep else None, xt.scales.ptr if keep else None, work.ptr, work.nbytes,
                               None), "mx4_linear")
    check(lib().bsq_stream_synchronize(None), "sync")
    y = out.download(_TYPE_NUMPY[out_type], m * w.rows).reshape(m, w.rows)
    return (y, xt) if keep else y


def mx4_linear_backward(dy: np.ndarray, xt: Mx4, wt: Mx4, type: int = TYPE_F32, g_type: int = TYPE_F32):
    """(dx, dw) of mx4_linear from the packed columns of x and of the weights."""
    dy = _typed(dy, type)
    _agree(dy.ndim == 2, "mx4_linear_backward: dy is a matrix")
    _agree(xt.batch == wt.batch == 1, "mx4_linear_backward: a batch of matrices")
    (m, n), k = dy.shape, wt.rows
    _agree(xt.cols == m, f"mx4_linear_backward: dy has {m} rows, the kept columns of x {xt.cols}")
    _agree(wt.cols == n, f"mx4_linear_backward: dy has {n} columns, the weights' columns {wt.cols}")
    _agree(xt.rows == k, f"mx4_linear_backward: x has {xt.rows} inputs, the weights {k}")
    if m == 0 or n == 0:  # an empty batch: the call itself wants one to sum over
        return np.zeros((m, k), _TYPE_NUMPY[g_type]), np.zeros((n, k), _TYPE_NUMPY[g_type])
    size = _TYPE_NUMPY[g_type].itemsize
    d, dx, dw = DeviceBuffer.from_array(dy), DeviceBuffer(m * k * size), DeviceBuffer(n * k * size)
    work = DeviceBuffer(workspace("bsq_mx4_linear_backward_workspace", m, n, k))
    check(lib().bsq_mx4_linear_backward(d.ptr, type, m, n, n, xt.codes.ptr, xt.scales.ptr, wt.codes.ptr, wt.scales.ptr,
                                        k, dx.ptr, k, dw.ptr, k, g_type, work.ptr, work.nbytes, None),
          "mx4_linear_backward")
    check(lib().bsq_stream_synchronize(None), "sync")
    return (dx.download(_TYPE_NUMPY[g_type], m * k).reshape(m, k), dw.download(_TYPE_NUMPY[g_type], n * k).reshape(n, k))


def moe_route(logits: np.ndarray, k: int, type: int = TYPE_F32, bias: np.ndarray | None = None,
              scoring: int = SCORE_SOFTMAX, groups: int = 1, kept: int = 1, renormalise: bool = True, scale: float = 1.0):
    """(ids, weights), tokens x k."""
    logits = _typed(logits, type)
    _agree(logits.ndim == 2, "moe_route: the logits are a matrix")
    tokens, experts = logits.shape
    _agree(bias is None or np.shape(bias) == (experts,), f"moe_route: a bias for each of {experts} experts")
    d = DeviceBuffer.from_array(logits)
    db = DeviceBuffer.from_array(np.ascontiguousarray(bias, np.float32)) if bias is not None else None
    ids, weights = DeviceBuffer(tokens * k * 4), DeviceBuffer(tokens * k * 4)
    check(lib().bsq_moe_route(d.ptr, type, tokens, experts, experts, db.ptr if db else None, scoring, groups, kept, k,
                              int(renormalise), scale, ids.ptr, weights.ptr, None), "moe_route")
    check(lib().bsq_stream_synchronize(None), "sync")
    return (ids.download(np.int32, tokens * k).reshape(tokens, k),
            weights.download(np.float32, tokens * k).reshape(tokens, k))


def moe_route_backward(logits: np.ndarray, ids: np.ndarray, d_weights: np.ndarray, type: int = TYPE_F32,
                       scoring: int = SCORE_SOFTMAX, renormalise: bool = True, scale: float = 1.0) -> np.ndarray:
    logits, ids = _typed(logits, type), np.ascontiguousarray(ids, np.int32)
    _agree(logits.ndim == 2, "moe_route_backward: the logits are a matrix")
    _agree(ids.ndim == 2 and len(ids) == len(logits), f"moe_route_backward: ids of {len(logits)} tokens")
    _agree(np.shape(d_weights) == ids.shape, "moe_route_backward: a gradient of weights for every id")
    (tokens, experts), k = logits.shape, ids.shape[1]
    d, di = DeviceBuffer.from_array(logits), DeviceBuffer.from_array(ids)
    dw, out = DeviceBuffer.from_array(np.ascontiguousarray(d_weights, np.float32)), DeviceBuffer(logits.nbytes)
    check(lib().bsq_moe_route_backward(d.ptr, type, tokens, experts, experts, scoring, k, int(renormalise), scale, di.ptr,
                                       dw.ptr, out.ptr, experts, None), "moe_route_backward")
    check(lib().bsq_stream_synchronize(None), "sync")
    return out.download(logits.dtype, tokens * experts).reshape(tokens, experts)


def moe_plan(ids: np.ndarray, experts: int):
    """(offsets, order) of the pairs in the experts' order."""
    ids = np.ascontiguousarray(ids, np.int32)
    d, off, order = DeviceBuffer.from_array(ids), DeviceBuffer(4 * (experts + 1)), DeviceBuffer(4 * ids.size)
    check(lib().bsq_moe_plan(d.ptr, ids.size, experts, off.ptr, order.ptr, None), "moe_plan")
    check(lib().bsq_stream_synchronize(None), "sync")
    return off.download(np.int32, experts + 1), order.download(np.int32, ids.size)


class MoeLinear:
    """The experts' layer on packed weights: forward(), then backward() of it."""

    def __init__(self, w: Mx4, wt: Mx4 | None = None):
        """w: a batch of n x inputs; wt: the batch of its columns (inputs x n),
        for the gradient of x."""
        _agree(wt is None or (wt.batch, wt.rows, wt.cols) == (w.batch, w.cols, w.rows),
               "MoeLinear: wt are the weights' columns, experts x inputs x n")
        self.done = False  # a forward call has left what backward() reads
        self.w, self.wt, self.experts, self.n, self.inputs = w, wt, w.batch, w.rows, w.cols

    def forward(self, x, ids, weights, type: int = TYPE_F32, out_type: int = TYPE_F32, y_type: int = TYPE_F32):
        self.done = False
        x, ids, weights = _typed(x, type), np.ascontiguousarray(ids, np.int32), np.ascontiguousarray(weights, np.float32)
        _agree(x.ndim == 2, "MoeLinear: x is a matrix")
        _agree(x.shape[1] == self.inputs, f"MoeLinear: x has {x.shape[1]} columns, the weights {self.inputs}")
        _agree(ids.ndim == 2 and len(ids) == len(x), f"MoeLinear: ids of {len(x)} tokens")
        _agree(weights.shape == ids.shape, "MoeLinear: routing weights for every id")
        m, k, e, n = len(x), ids.shape[1], self.experts, self.n
        self.type, self.m, self.k, self.y_type = type, m, k, y_type
        self.x, self.ids, self.weights = (DeviceBuffer.from_array(v) for v in (x, ids, weights))
        self.offsets, self.order = DeviceBuffer(4 * (e + 1)), DeviceBuffer(4 * m * k)
        self.y = DeviceBuffer(m * k * n * _TYPE_NUMPY[y_type].itemsize)
        out = DeviceBuffer(m * n * _TYPE_NUMPY[out_type].itemsize)
        work = DeviceBuffer(workspace("bsq_moe_linear_workspace", m, k, n, self.inputs, e))
        check(lib().bsq_moe_linear(self.x.ptr, type, m, self.inputs, self.inputs, self.ids.ptr, self.weights.ptr, k,
                                   self.w.codes.ptr, self.w.scales.ptr, e, n, self.offsets.ptr, self.order.ptr,
                                   self.y.ptr, y_type, out.ptr, out_type, n, work.ptr, work.nbytes, None), "moe_linear")
        check(lib().bsq_stream_synchronize(None), "sync")
        self.done = True
        return out.download(_TYPE_NUMPY[out_type], m * n).reshape(m, n)

    def backward(self, d_out, type: int = TYPE_F32, g_type: int = TYPE_F32):
        """(dx, d weights, dw)."""
        d_out = _typed(d_out, type)
        _agree(self.done, "MoeLinear: backward() goes back through a forward() call")
        _agree(self.wt is not None, "MoeLinear: backward() needs the weights' columns")
        _agree(d_out.ndim == 2, "MoeLinear: d_out is a matrix")
        _agree(d_out.shape == (self.m, self.n), f"MoeLinear: d_out is {self.m} x {self.n}")
        m, k, n, e, inputs = self.m, self.k, self.n, self.experts, self.inputs
        t = _TYPE_NUMPY[g_type]
        d, dx, dw = DeviceBuffer.from_array(d_out), DeviceBuffer(m * inputs * t.itemsize), DeviceBuffer(e * n * inputs * t.itemsize)
        dweights = DeviceBuffer(4 * m * k)
        work = DeviceBuffer(workspace("bsq_moe_linear_backward_workspace", m, k, n, inputs, e))
        check(lib().bsq_moe_linear_backward(d.ptr, type, m, n, n, self.x.ptr, self.type, inputs, inputs, self.ids.ptr,
                                            self.weights.ptr, k, self.offsets.ptr, self.order.ptr, self.y.ptr,
                                            self.y_type, self.wt.codes.ptr, self.wt.scales.ptr, e, dx.ptr, inputs,
                                            dweights.ptr, dw.ptr, g_type, work.ptr, work.nbytes, None),
              "moe_linear_backward")
        check(lib().bsq_stream_synchronize(None), "sync")
        return (dx.download(t, m * inputs).reshape(m, inputs), dweights.download(np.float32, m * k).reshape(m, k),
                dw.download(t, e * n * inputs).reshape(e, n, inputs))
