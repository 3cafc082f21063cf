/*
 * bitsqz_llm C-ABI boundary -- MI355X (gfx950).
 *
 * Plain extern "C" entry points (plain pointers and sizes, no HIP or torch
 * types) for FFI callers: Python ctypes, cgo, JNI, N-API.  Device pointers are
 * passed as ordinary pointers; `stream` is a hipStream_t passed as void*
 * (NULL = the HIP null stream).  Every int-returning function returns 0 on
 * success and 1 on failure (the reference convention, src/bitsqz_llm.cu);
 * bsq_last_error() returns the message of the most recent failure on the
 * calling thread.
 *
 * Three groups:
 *   1. bsq_*          -- extern "C" twins of the nine C++-linkage ABI
 *                        functions in bitsqz_llm.hpp (same semantics).
 *   2. bsq_device_*   -- the same compress / decompress pipeline with the
 *                        packed sections kept in device memory (no host
 *                        round trip, no host synchronisation); used to measure
 *                        the device-resident path and by the host ABI itself.
 *   3. bsq_topk_*, bsq_quant_*, bsq_svd_*, bsq_reconstruct_* -- the four
 *                        module operators the pipeline is built from, each
 *                        mirroring a reference module entry point.
 * and beside them memory helpers (4), the legacy formats (5), and layers that
 * compute on 4-bit matrices (6: bsq_mx4_*, bsq_moe_*).
 */
#ifndef BITSQZ_LLM_C_H
#define BITSQZ_LLM_C_H

#include <stdint.h>

#include "bitsqz_llm.hpp"

#ifdef __cplusplus
extern "C" {
#endif

#define BSQ_API __attribute__((visibility("default")))

/* ---------------------------------------------------------------------------
 * 0. Diagnostics
 * ------------------------------------------------------------------------- */

/* Message of the last failure on this thread ("" if none).  No reference
 * counterpart: the reference discards exception messages at the boundary
 * (src/bitsqz_llm.cu:878-881). */
BSQ_API const char *bsq_last_error(void);

/* Library version string. */
BSQ_API const char *bsq_version(void);

/* ---------------------------------------------------------------------------
 * 1. extern "C" twins of the C++ ABI (include/bitsqz_llm.hpp)
 * ------------------------------------------------------------------------- */

/* replaces bitsqz_llm_compress_initialize, reference bitsqz_llm.hpp:95-105 */
BSQ_API int bsq_compress_initialize(uint16_t num_rows, uint16_t num_columns,
                                    float outlier_topk_ratio, float error_correction_topk_ratio,
                                    int svd_ranks, int svd_niters,
                                    int svd_uv_format, int svd_s_format,
                                    int quantization_only_format, int input_location);
/* replaces bitsqz_llm_compress_release, reference bitsqz_llm.hpp:107 */
BSQ_API void bsq_compress_release(void);
/* replaces bitsqz_llm_decompress_initialize, reference bitsqz_llm.hpp:109-117 */
BSQ_API int bsq_decompress_initialize(uint16_t num_rows, uint16_t num_columns,
                                      float outlier_topk_ratio, float error_correction_topk_ratio,
                                      int svd_ranks, int svd_uv_format, int svd_s_format,
                                      int quantization_only_format);
/* replaces bitsqz_llm_decompress_release, reference bitsqz_llm.hpp:119 */
BSQ_API void bsq_decompress_release(void);
/* replaces bitsqz_llm_compress, reference bitsqz_llm.hpp:121-124 */
BSQ_API int bsq_compress(const float *row_major_matrix_float_data, bitsqz_llm_array_t **out,
                         bitsqz_llm_compress_profile_t *profile);
/* replaces bitsqz_llm_decompress, reference bitsqz_llm.hpp:132-135 */
BSQ_API int bsq_decompress(const bitsqz_llm_array_t *compressed, float *d_dst,
                           uint32_t dst_num_elements);
/* replaces bitsqz_llm_get_packed_size, reference bitsqz_llm.hpp:137 */
BSQ_API uint64_t bsq_get_packed_size(const bitsqz_llm_array_t *compressed);
/* replaces load_bitsqz_llm_from_buffer, reference bitsqz_llm.hpp:139 */
BSQ_API bitsqz_llm_array_t *bsq_load_from_buffer(const void *buffer, uint64_t buffer_size);
/* replaces bitsqz_llm_free, reference bitsqz_llm.hpp:141 */
BSQ_API void bsq_free(bitsqz_llm_array_t *compressed);

/* Test hook: replace the Gaussian sketch of the compress runtime's SVD by a
 * caller-supplied device matrix (N_work x rank, row-major, N_work =
 * min(rows, cols)); NULL restores the built-in generator.  The reference
 * draws the sketch from cuRAND inside a CUDA graph
 * (modules/svd_lowrank_cuda/src/svd_lowrank_cuda.cu:289-291, 552-556), which
 * no other implementation can reproduce, so parity of the SVD path is defined
 * with an injected sketch.  The pointer must stay valid while it is set. */
BSQ_API int bsq_compress_set_sketch(const float *d_sketch);

/* ---------------------------------------------------------------------------
 * 2. Device-resident pipeline
 * ------------------------------------------------------------------------- */

/* A packed object whose sections live in device memory.  `header` carries the
 * header fields the host object would have (section offsets/sizes are
 * payload-relative, `payload` is NULL) with the flags the host can decide
 * (SVD, outlier).  Whether the error-correction section is present is decided
 * on the device: the word *d_flags (device memory) has bit 2 set when it is,
 * and header.section_error_topk describes it for that case.  The component
 * pointers are device pointers owned by the compress runtime; they stay valid
 * until the next compress call or release.  For quantised sections d_dense is
 * NULL and the scales / codes pointers are set; for FP32 sections d_dense is
 * set. */
typedef struct {
    bitsqz_llm_array_t header;
    const uint32_t *d_flags;
    /* quantised / dense sections: U, S, V, direct (index 0..3) */
    const float *d_dense[4];        /* FP32 storage (section stored dense) */
    const float *d_scales_f32[4];   /* NF4 block scales                      */
    const uint8_t *d_scales_u8[4];  /* NF4_DQ E4M3 block scale codes         */
    const float *d_dq_scale[4];     /* NF4_DQ global scale (1 float)         */
    const uint8_t *d_codes[4];      /* packed nibbles                        */
    uint64_t count[4];              /* element count of each section         */
    /* top-k sections: outlier (0), error (1) */
    const uint16_t *d_topk_idx[2];
    const float *d_topk_val[2];
    uint16_t topk_k[2];
} bsq_device_packed_t;

/* Run the whole compress pipeline of the initialised compress runtime on
 * `d_input` (device memory, row-major rows x cols), enqueued on the runtime's
 * stream; returns without a host synchronisation. */
BSQ_API int bsq_device_compress(const float *d_input, bsq_device_packed_t *out);

/* Decode a device-resident packed object into `d_dst` with the initialised
 * decompress runtime (same configuration checks as bsq_decompress), enqueued
 * on the compress runtime's stream when one exists; no host synchronisation. */
BSQ_API int bsq_device_decompress(const bsq_device_packed_t *packed, float *d_dst,
                                  uint32_t dst_num_elements);

/* Wait for all work the runtimes enqueued. */
BSQ_API int bsq_device_synchronize(void);

/* The stream the runtimes enqueue on (a hipStream_t). */
BSQ_API void *bsq_runtime_stream(void);

/* Lanes (no counterpart in the reference, whose runtimes are process-global
 * singletons, src/bitsqz_llm.cu:33-138): `lanes` (1..8) independent pairs of
 * compress + decompress runtimes with the given configuration (DEVICE input;
 * the decompress runtime takes the effective rank), each on its own stream.
 * bsq_lanes_roundtrip enqueues one device-resident compress of d_input and
 * the decompress of its result into d_dst (rows x cols floats) on the lane's
 * stream, exactly as bsq_device_compress + bsq_device_decompress do, and
 * returns without a host synchronisation.  Lanes share no buffers, so round
 * trips on different lanes run concurrently; a lane's packed object lives
 * until its next round trip.  For callers with several matrices in flight
 * (e.g. the activations of several layers). */
BSQ_API int bsq_lanes_initialize(int lanes, uint16_t rows, uint16_t cols, float outlier_topk_ratio,
                                 float error_correction_topk_ratio, int svd_ranks, int svd_niters,
                                 int svd_uv_format, int svd_s_format, int quantization_only_format);
BSQ_API int bsq_lanes_roundtrip(int lane, const float *d_input, float *d_dst);
BSQ_API void *bsq_lanes_stream(int lane);
BSQ_API int bsq_lanes_synchronize(void);
BSQ_API void bsq_lanes_release(void);

/* ---------------------------------------------------------------------------
 * 3. Module operators
 * ------------------------------------------------------------------------- */

/* k = roundf(cols * ratio), clamped to [1, cols] when ratio > 0.
 * replaces topk_compute_num_topk_columns, reference
 * modules/topk_cuda/src/topk_cuda.cu:53-69 (which throws on a bad ratio;
 * here: returns 1). */
BSQ_API int bsq_topk_num_columns(uint16_t num_columns, float ratio, uint16_t *out_k);

/* Per-row top-k of |x| (NaN ranks lowest), ordered by |x| descending with
 * ties to the lower column; writes indices[r*k + j] and the signed values.
 * If d_residual is not NULL it receives the input with the selected entries
 * zeroed (it may alias d_input: in-place separation).
 * replaces topk_extraction / topk_separation, reference
 * modules/topk_cuda/src/topk_cuda.cu:186-201. */
BSQ_API int bsq_topk_select(const float *d_input, uint16_t rows, uint16_t cols, uint16_t k,
                            uint16_t *d_indices, float *d_values, float *d_residual,
                            void *stream);

/* dense[r, idx] += value for every entry (topk_apply, reference
 * modules/topk_cuda/src/topk_cuda.cu:221-233) or, with accumulate == 0,
 * dense = 0 then dense[r, idx] = value (topk_decompress, :203-219). */
BSQ_API int bsq_topk_scatter(const uint16_t *d_indices, const float *d_values, uint16_t rows,
                             uint16_t cols, uint16_t k, float *d_dense, int accumulate,
                             void *stream);

/* NF4 (method 11) or NF4_DQ (method 10) block-64 quantisation of `count`
 * floats.  NF4 writes d_scales_f32[ceil(count/64)]; NF4_DQ writes
 * d_scales_u8[ceil(count/64)] and *d_dq_scale.  Codes: ceil(count/2) bytes.
 * replaces quantization_cuda_compress, reference
 * modules/quantization_cuda/src/quantization_cuda.cu:564-624. */
BSQ_API int bsq_quant_compress(const float *d_input, uint64_t count, int method,
                               float *d_scales_f32, uint8_t *d_scales_u8, float *d_dq_scale,
                               uint8_t *d_codes, void *stream);

/* replaces quantization_cuda_decompress, reference
 * modules/quantization_cuda/src/quantization_cuda.cu:626-663. */
BSQ_API int bsq_quant_decompress(uint64_t count, int method, const float *d_scales_f32,
                                 const uint8_t *d_scales_u8, const float *d_dq_scale,
                                 const uint8_t *d_codes, float *d_output, void *stream);

/* Test hooks for the scalar codec primitives (reference
 * quantization_cuda.cu:43-128): NF4 nearest-code of each value, E4M3 encode of
 * each value, E4M3 decode of each code. */
BSQ_API int bsq_quant_nf4_codes(const float *d_values, uint64_t n, uint8_t *d_codes, void *stream);
BSQ_API int bsq_quant_e4m3_encode(const float *d_values, uint64_t n, uint8_t *d_codes, void *stream);
BSQ_API int bsq_quant_e4m3_decode(const uint8_t *d_codes, uint64_t n, float *d_values, void *stream);

/* NF4 code of every float bit pattern in [lo, hi) (hi <= 2^32): 16-bin
 * histogram and sum over patterns of code * (pattern mod 65521), written to
 * device memory; pins the device code function against a CPU sweep. */
BSQ_API int bsq_quant_nf4_code_sweep(uint64_t lo, uint64_t hi, unsigned long long *d_hist16,
                                     unsigned long long *d_checksum, void *stream);
/* The 15 exact decision thresholds the device NF4 code function uses for
 * |v| < 2 (code = number of thresholds <= v). */
BSQ_API void bsq_nf4_thresholds(float out[15]);

/* Randomised rank-q SVD of a row-major m x n matrix with `niter` power
 * iterations and no oversampling: U (m x q), S (q), V (n x q), row-major,
 * q = max(1, min(q, m, n)).  d_sketch (min(m,n) x q, row-major) may be NULL
 * to draw the sketch from the built-in generator with `seed`.
 * replaces svd_lowrank_cuda, reference
 * modules/svd_lowrank_cuda/src/svd_lowrank_cuda.cu:541-581. */
BSQ_API int bsq_svd_lowrank(const float *d_A, int m, int n, int q, int niter,
                            const float *d_sketch, uint64_t seed, float *d_U, float *d_S,
                            float *d_V, void *stream);

/* bsq_svd_lowrank without any device allocation.  No counterpart in the
 * reference: for callers that cannot allocate device memory (code under HIP
 * graph capture, allocation-free serving loops).  Same arguments and results
 * as bsq_svd_lowrank (the same kernels on the same plan layout), but the
 * plan's buffers are carved from the library's fixed 256 MiB device array
 * (one copy per GPU, held until the process ends), so shapes whose plan needs
 * more return 1 with the byte counts in bsq_last_error().  Asynchronous on
 * `stream` (no synchronisation); calls that overlap on one GPU share that
 * array and race. */
BSQ_API int bsq_svd_lowrank_noalloc(const float *d_A, int m, int n, int q, int niter,
                                    const float *d_sketch, uint64_t seed, float *d_U,
                                    float *d_S, float *d_V, void *stream);

/* out (m x n, row-major) = U (m x k) * diag(S) * V (n x k)^T.
 * replaces reconstruct_lowrank_cuda, reference
 * modules/reconstruct_lowrank_cuda/src/reconstruct_lowrank_cuda.cu:21-62,153-171. */
BSQ_API int bsq_reconstruct_lowrank(const float *d_U, const float *d_S, const float *d_V, int m,
                                    int n, int k, float *d_out, void *stream);

/* Fill `n` floats with N(0,1) draws of the built-in sketch generator
 * (counter-based Philox4x32-10 + Box-Muller; deterministic in (seed, index)). */
BSQ_API int bsq_gaussian_fill(float *d_out, uint64_t n, uint64_t seed, void *stream);

/* ---------------------------------------------------------------------------
 * 4. Device memory helpers for FFI callers without a GPU framework (no
 *    reference counterpart; thin wrappers over hipMalloc / hipMemcpy).
 * ------------------------------------------------------------------------- */
BSQ_API int bsq_device_count(int *count);
BSQ_API int bsq_device_malloc(void **ptr, uint64_t bytes);
BSQ_API int bsq_device_free(void *ptr);
BSQ_API int bsq_memcpy_h2d(void *dst, const void *src, uint64_t bytes);
BSQ_API int bsq_memcpy_d2h(void *dst, const void *src, uint64_t bytes);
BSQ_API int bsq_memcpy_d2d(void *dst, const void *src, uint64_t bytes);
BSQ_API int bsq_device_memset(void *dst, int value, uint64_t bytes);
/* Pinned (page-locked) host memory, hipHostMalloc / hipHostFree, and an
 * asynchronous host-to-device copy on a caller-chosen stream (null: the
 * default stream). */
BSQ_API int bsq_host_malloc(void **ptr, uint64_t bytes);
BSQ_API int bsq_host_free(void *ptr);
BSQ_API int bsq_memcpy_h2d_async(void *dst, const void *src, uint64_t bytes, void *stream);
BSQ_API int bsq_stream_synchronize(void *stream);
/* HIP events on a caller-chosen stream (timing without a GPU framework). */
BSQ_API int bsq_event_create(void **event);
BSQ_API int bsq_event_destroy(void *event);
BSQ_API int bsq_event_record(void *event, void *stream);
BSQ_API int bsq_event_elapsed_ms(void *start, void *stop, float *ms);

/* Instrumentation (no counterpart in the reference): while started, the
 * launches of six classes inside the compress / decompress pipelines are
 * bracketed by HIP events on their own stream.  _stop waits for those events
 * and returns the summed time and launch count of the low-rank reconstruction
 * GEMMs; _read then returns any class: 0 = reconstruction GEMM, 1 = the range
 * finder's products with the big matrix (split-K / stream-K reductions
 * included), 2 = outlier separation top-k, 3 = error-correction top-k,
 * 4 = direct-section encode (with the NF4_DQ global-scale reduce),
 * 5 = direct-section decode (with the fused top-k scatter). */
BSQ_API int bsq_kernel_timer_start(void);
BSQ_API int bsq_kernel_timer_read(int timer_class, double *total_ms, int *launches);
/* Plain device copy kernel (16 bytes per lane), the known-size reference for
 * calibrating HBM byte counters.  bytes and both pointers 16-byte aligned. */
BSQ_API int bsq_copy_kernel(const void *d_src, void *d_dst, uint64_t bytes, void *stream);
BSQ_API int bsq_kernel_timer_stop(double *total_ms, int *launches);

/* ---------------------------------------------------------------------------
 * 5. Legacy quantisation formats (include/quantization.hpp): the reference's
 *    CPU codec dispatcher, here encoding and decoding on the GPU.
 * ------------------------------------------------------------------------- */
/* extern "C" twins of the five C++-linkage functions of include/quantization.hpp;
 * replace quantization_compress / quantization_decompress /
 * quantization_get_packed_size / load_quantization_from_buffer /
 * quantization_free, reference
 * legacy_modules/quantization/src/quantization.cpp:125-489.  `method` is a
 * quantization_method_t value; buffers are quantization_buffer_t *. */
BSQ_API int bsq_legacy_compress(int method, const float *src, uint64_t n, void **out);
BSQ_API int bsq_legacy_decompress(const void *buf, float *dst, uint64_t n);
BSQ_API long long bsq_legacy_packed_size(const void *buf);
BSQ_API void *bsq_legacy_load(const void *buffer, long long size);
BSQ_API void bsq_legacy_free(void *buf);

/* Bytes of the payload (format struct + arrays) of n elements, or -1.  The
 * reference's get_*_array_size (e.g. q8_0_impl.cpp:3-6) on the struct that
 * its compress writes. */
BSQ_API long long bsq_legacy_payload_bytes(int method, uint64_t n);

/* Device-resident codec (no reference counterpart: the reference codecs take
 * host arrays).  Encode writes the payload image of n device floats to
 * d_payload (16-byte aligned, bsq_legacy_payload_bytes bytes): the format
 * struct with its counts and scale, then its arrays, byte-identical to the
 * reference's payload except the struct's pointer fields, which are left
 * unspecified (FP8, FP4, NVFP4 and NF4_DQ use one as reduction scratch).
 * Decode reads such an image of n elements.  Asynchronous on `stream`. */
BSQ_API int bsq_legacy_encode_device(int method, const float *d_src, uint64_t n, void *d_payload,
                                     void *stream);
BSQ_API int bsq_legacy_decode_device(int method, const void *d_payload, uint64_t n, float *d_dst,
                                     void *stream);

/* Test hook: adds to *d_checksum the sum over float patterns p in [lo, hi)
 * (hi <= 2^32) of (r(p) + 1) * (p mod 65521), where r is the device FP16
 * conversion (kind 0), BF16 conversion (1) or MX block exponent as a byte
 * (2: max norm 448, 3: max norm 6). */
BSQ_API int bsq_legacy_sweep(int kind, uint64_t lo, uint64_t hi, unsigned long long *d_checksum,
                             void *stream);

/* ---------------------------------------------------------------------------
 * 6. Microscaled 4-bit matrices (MX4) and layers that compute with them (no
 *    reference counterpart: its MXFP4 stores flat arrays and only decodes).
 *
 *    A packed matrix of rows x cols: blocks of 32 values along a row share a
 *    power of two, the smallest 2^e, e >= -126, with no value above 6 times it;
 *    a value over it is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6
 *    (ties to the even code) and its sign, E2M1.  A block that holds a NaN or an
 *    infinity is NaN as a whole.  Row-major codes, two a byte with the first in
 *    the low half, and row-major scale bytes (e + 127; 255: NaN); rows padded
 *    with zeros to a multiple of 256 values.  Codes are 16-byte and scales
 *    8-byte aligned (so is a workspace, 16).
 *
 *    Element types: 0 FP32, 1 BF16, 2 FP16.  `ld` counts elements from one row
 *    to the next.  Sums are held in FP32 (in the order of the matrix
 *    instructions, the tiles and the splits: the same from run to run) and
 *    rounded once; the join of experts sums y as it is stored.  All calls are
 *    asynchronous on `stream`, keep nothing between calls and take their
 *    workspace from the caller (its bytes: the function beside them), so they
 *    can be captured, and run on several streams with a workspace each.  The
 *    workspace functions give UINT64_MAX, with the reason in bsq_last_error(),
 *    for sizes that the call refuses, or without a device where the size hangs
 *    on its CUs.
 * ------------------------------------------------------------------------- */
BSQ_API uint64_t bsq_mx4_codes_bytes(uint64_t rows, uint64_t cols);
BSQ_API uint64_t bsq_mx4_scales_bytes(uint64_t rows, uint64_t cols);

/* Packs `batch` matrices of rows x cols (`stride` elements apart): their rows
 * into d_codes / d_scales, and / or their columns, as the packed cols x rows
 * transposes, into d_codes_t / d_scales_t, from one read.  Either pair may be
 * NULL.  The batch's packed matrices follow one another. */
BSQ_API int bsq_mx4_encode(const void *d_x, int type, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t ld,
                           uint64_t stride, uint8_t *d_codes, uint8_t *d_scales, uint8_t *d_codes_t,
                           uint8_t *d_scales_t, void *stream);
BSQ_API int bsq_mx4_decode(const uint8_t *d_codes, const uint8_t *d_scales, uint64_t rows, uint64_t cols, void *d_out,
                           int type, uint64_t ld, void *stream);

/* out (m x n) = A B^T of packed A (m x k) and B (n x k). */
BSQ_API uint64_t bsq_mx4_product_workspace(uint64_t m, uint64_t n, uint64_t k);
BSQ_API int bsq_mx4_product(const uint8_t *d_a_codes, const uint8_t *d_a_scales, uint64_t m, const uint8_t *d_b_codes,
                            const uint8_t *d_b_scales, uint64_t n, uint64_t k, void *d_out, int type, uint64_t ld,
                            void *d_work, uint64_t work_bytes, void *stream);

/* A dense layer: out (m x n) = q(x) W^T, x (m x k) packed on the way, W packed
 * (n x k).  With d_xt_codes / d_xt_scales (may be NULL) the packed k x m
 * transpose of x is kept for the backward pass: the activations at 4.25 bits a
 * value. */
BSQ_API uint64_t bsq_mx4_linear_workspace(uint64_t m, uint64_t n, uint64_t k);
BSQ_API int bsq_mx4_linear(const void *d_x, int x_type, uint64_t m, uint64_t k, uint64_t ldx, const uint8_t *d_w_codes,
                           const uint8_t *d_w_scales, uint64_t n, void *d_out, int out_type, uint64_t ldo,
                           uint8_t *d_xt_codes, uint8_t *d_xt_scales, void *d_work, uint64_t work_bytes, void *stream);
/* Its gradients, straight through the rounding: dx (m x k) = q(dy) W with the
 * weights' columns d_wt_* (k x n packed), dw (n x k) = q(dy^T) q(x^T)^T with
 * the columns of x that the forward call kept.  d_dx or d_dw may be NULL.  m
 * and n are at least 1: unlike the forward call it refuses an empty batch, whose
 * dw, all zeros, is the caller's to write. */
BSQ_API uint64_t bsq_mx4_linear_backward_workspace(uint64_t m, uint64_t n, uint64_t k);
BSQ_API int bsq_mx4_linear_backward(const void *d_dy, int type, uint64_t m, uint64_t n, uint64_t ldy,
                                    const uint8_t *d_xt_codes, const uint8_t *d_xt_scales, const uint8_t *d_wt_codes,
                                    const uint8_t *d_wt_scales, uint64_t k, void *d_dx, uint64_t lddx, void *d_dw,
                                    uint64_t lddw, int g_type, void *d_work, uint64_t work_bytes, void *stream);

/* Routing of tokens to k of `experts` (up to 1024; k up to 64) from their
 * logits.  Scores: softmax over the experts (scoring 0) or sigmoid (1).  The
 * choice goes by the logits, or by score + d_bias[expert] where d_bias is not
 * NULL; with groups > 1 (equal runs of experts, up to 64 groups) only among the
 * `kept` groups whose largest entry, or with a bias whose two largest entries'
 * sum, is largest; ties go to the lowest number.  An expert whose logit is NaN
 * or at or below its type's lowest finite value is closed to the token.  ids:
 * tokens x k, best first, -1 (weight 0) where no open expert is left; weights:
 * the scores, over their sum if `renormalise` (over the smallest normal FP32
 * number where the sum is below it), times `scale`. */
BSQ_API int bsq_moe_route(const void *d_logits, int type, uint64_t tokens, uint32_t experts, uint64_t ld,
                          const float *d_bias, int scoring, uint32_t groups, uint32_t kept, uint32_t k, int renormalise,
                          float scale, int32_t *d_ids, float *d_weights, void *stream);
/* d logits (of the logits' type) from d weights and the ids of the choice. */
BSQ_API int bsq_moe_route_backward(const void *d_logits, int type, uint64_t tokens, uint32_t experts, uint64_t ld,
                                   int scoring, uint32_t k, int renormalise, float scale, const int32_t *d_ids,
                                   const float *d_d_weights, void *d_d_logits, uint64_t ldd, void *stream);
/* The pairs (token, place) = (p / k, p % k) in the experts' order: expert e's
 * are d_order[d_offsets[e] .. d_offsets[e + 1]), ascending; pairs whose id is
 * not an expert follow the last.  d_offsets: experts + 1 entries. */
BSQ_API int bsq_moe_plan(const int32_t *d_ids, uint64_t pairs, uint32_t experts, int32_t *d_offsets, int32_t *d_order,
                         void *stream);
/* out[t] = sum over the token's experts of weight * y[t k + j] (y: tokens k x n,
 * rows side by side). */
BSQ_API int bsq_moe_combine(const void *d_y, int y_type, uint64_t tokens, uint32_t k, uint64_t n, const int32_t *d_ids,
                            const float *d_weights, uint32_t experts, void *d_out, int type, uint64_t ld, void *stream);

/* The experts' layer: y[t k + j] = q(x[t]) W_e^T for e = ids[t k + j] and out =
 * the join of y by the weights.  W: experts packed matrices of n x inputs, one
 * after another.  d_offsets, d_order (as bsq_moe_plan) and d_y (tokens k x n;
 * zero rows where a pair has no expert) are written and serve the backward
 * pass.  out and the gradient of the weights are as fine as y's type, which is
 * the caller's choice: FP32 y leaves out one rounding, BF16 y halves the bytes
 * and rounds each pair's product once more (0.0024 in place of 0.0017 of a BF16
 * out), FP16 y is infinite above 65504.  Gradients by the backward call sum FP32
 * products whatever their type. */
BSQ_API uint64_t bsq_moe_linear_workspace(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs, uint32_t experts);
BSQ_API int bsq_moe_linear(const void *d_x, int x_type, uint64_t tokens, uint64_t inputs, uint64_t ldx,
                           const int32_t *d_ids, const float *d_weights, uint32_t k, const uint8_t *d_w_codes,
                           const uint8_t *d_w_scales, uint32_t experts, uint64_t n, int32_t *d_offsets, int32_t *d_order,
                           void *d_y, int y_type, void *d_out, int out_type, uint64_t ldo, void *d_work,
                           uint64_t work_bytes, void *stream);
/* Its gradients, each optional (NULL): dx = sum of weight * q(d out) W_e with
 * the weights' columns d_wt_* (experts packed matrices of inputs x n), d
 * weights[t, j] = <d out[t], y[t k + j]>, dw (experts x n x inputs) = the sum
 * over the expert's pairs of q(weight d out)^T q(x), in blocks of 32 pairs (up
 * to some 33 million pairs: tokens k / 256 + experts <= 2^17). */
BSQ_API uint64_t bsq_moe_linear_backward_workspace(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs,
                                                   uint32_t experts);
BSQ_API int bsq_moe_linear_backward(const void *d_d_out, int d_type, uint64_t tokens, uint64_t n, uint64_t ldd,
                                    const void *d_x, int x_type, uint64_t inputs, uint64_t ldx, const int32_t *d_ids,
                                    const float *d_weights, uint32_t k, const int32_t *d_offsets, const int32_t *d_order,
                                    const void *d_y, int y_type, const uint8_t *d_wt_codes, const uint8_t *d_wt_scales,
                                    uint32_t experts, void *d_dx, uint64_t lddx, float *d_d_weights, void *d_dw,
                                    int g_type, void *d_work, uint64_t work_bytes, void *stream);

/* ---------------------------------------------------------------------------
 * 7. Attention over a paged cache of keys and values in MX4, rotary positions
 *    and a step's bookkeeping (no reference counterpart).
 *
 *    The cache: `pages` pages of `page` tokens.  A page holds, head after head
 *    of keys and values, the keys' codes, the values' codes, the keys' scales
 *    and the values' scales; a head's row is padded with zeros to whole blocks of
 *    32 values (B blocks).  Codes: a token's 16 B bytes, two codes a byte with the
 *    first in the low half, tokens side by side.  Scales, bytes as in group 6: 16
 *    tokens side by side (16 B bytes), in them that of token t and block b at
 *    4 (B (t % 4) + b) + t / 4.  A slot is page * page size + place in the page.
 *
 *    Whole numbers are int32.  As in group 6 all calls are asynchronous on
 *    `stream`, keep nothing between calls, take their workspace from the caller
 *    and can be captured; types, leading dimensions, returns and size queries are
 *    those of group 6 too.  Results may lie beside what a call reads, in other
 *    columns of rows of one distance; results on it are refused where the calls
 *    say so.  What device arrays hold is not checked by the host: page numbers and
 *    slots outside the cache, lengths outside the table and starts outside the
 *    tokens are left out by the kernels, as said below.
 * ------------------------------------------------------------------------- */
typedef struct {
    uint8_t *d_pages; /* bsq_kv4_cache_bytes bytes, 16-byte aligned */
    uint64_t pages;   /* pages * page < 2^31 */
    uint32_t page;    /* tokens of a page: 16, 32, 64, 128 or 256 */
    uint32_t heads;   /* of keys and values */
    uint32_t dim;     /* values of a head, 1 to 256 */
} bsq_kv4_cache_t;
BSQ_API uint64_t bsq_kv4_cache_bytes(uint64_t pages, uint32_t page, uint32_t heads, uint32_t dim);

/* A step's bookkeeping.  Request r holds d_lengths[r] tokens, in the pages of
 * its row of d_table (`width` entries), and gets d_new[r] more; below zero it
 * has ended.  d_free is a stack of free pages (room for all `pages`, the first
 * *d_free_count in use).  First the ended requests' pages go onto it, in the
 * order of requests and of their rows; then each request in turn takes the pages
 * that its new tokens need beyond those it holds, from the top, into its row.
 * A request is not served where the stack runs out (nor are those behind it that
 * need a page), its row is too short, or the tokens up to its last, those of the
 * requests before it among them, are more than `tokens`.
 * Written: d_lengths_out[r], the length with the new tokens (as it was where not
 * served, 0 where ended; may be d_lengths); d_left[0], the pages left on the
 * stack (d_left may be d_free_count), and d_left[1], the requests not served;
 * d_starts[0 .. requests], where each request's new tokens begin among the
 * `tokens` places; and for each place its request (d_requests, may be NULL), its
 * position and its slot: -1 behind the last token, position and slot also of
 * requests not served.  Up to 16384 requests; requests * width < 2^31. */
BSQ_API uint64_t bsq_kv4_plan_workspace(uint32_t requests);
BSQ_API int bsq_kv4_plan(const int32_t *d_lengths, const int32_t *d_new, uint32_t requests, int32_t *d_table,
                         uint32_t width, uint32_t page, int32_t *d_free, uint64_t pages, const int32_t *d_free_count,
                         int32_t *d_lengths_out, int32_t *d_left, int32_t *d_starts, uint64_t tokens,
                         int32_t *d_requests, int32_t *d_positions, int32_t *d_slots, void *d_work, uint64_t work_bytes,
                         void *stream);

/* Rotary positions: of a head's first `dims` values (even), pair i = (x[i],
 * x[i + dims / 2]), or (x[2 i], x[2 i + 1]) if `interleaved`, becomes factor
 * (a cos t - b sin t, b cos t + a sin t), t = position * d_frequencies[i]; the
 * others stay as they are.  Angles, sine and cosine are FP64; the pair's products
 * are FP64 for FP32 values and for keys that go into the cache, FP32 for other
 * 16-bit values; rounded through FP32 to the type. */
typedef struct {
    const double *d_frequencies; /* dims / 2 */
    uint32_t dims;
    int interleaved;
    float factor;
} bsq_rope_t;
/* Fills host arrays: frequencies base^(-2 i / dims), for contexts `stretch` times
 * `length`: scaling 0 as they are (stretch is not used); 1 all over stretch; 2
 * those of the base times stretch^(dims / (dims - 2)); 3 by parts: pairs that
 * turn over 32 times in `length` positions as they are, those that turn less
 * than once over stretch, a ramp between.  *factor: 1, for 3 it is
 * 1 + ln(stretch) / 10. */
BSQ_API int bsq_rope_frequencies(uint32_t dims, double base, int scaling, double stretch, double length,
                                 double *frequencies, float *factor);
/* out = x turned (`back`: turned back, times factor: the gradient of x from that
 * of out); tokens rows of `heads` heads side by side; out may be x, with its
 * rows, else it may not lie on them.  Rows whose position is below zero are left as
 * they are. */
BSQ_API int bsq_rope(const bsq_rope_t *rope, const int32_t *d_positions, const void *d_x, int type, uint64_t tokens,
                     uint32_t heads, uint32_t dim, uint64_t ldx, int back, void *d_out, uint64_t ldo, void *stream);

/* A step's tokens: queries (q_heads heads; d_q may be NULL) turned to d_q_out
 * (may be d_q, with its rows, else it may not lie on them; never on keys or
 * values), keys turned, rounded to their type and packed, values packed, both into
 * the cache at d_slots.  rope NULL: nothing is turned, and d_positions may be
 * NULL.  A token whose position is below zero is left out, one whose slot is
 * outside the cache leaves only its queries.  Where two tokens have one slot, it
 * holds parts of either. */
BSQ_API int bsq_kv4_append(const bsq_kv4_cache_t *cache, const bsq_rope_t *rope, const int32_t *d_positions,
                           const int32_t *d_slots, uint64_t tokens, int type, const void *d_q, uint32_t q_heads,
                           uint64_t ldq, void *d_q_out, uint64_t ldqo, const void *d_k, uint64_t ldk, const void *d_v,
                           uint64_t ldv, void *stream);
/* The keys and values at d_slots (either may be NULL; they may not lie on one
 * another); rows of slots outside the cache are left as they are. */
BSQ_API int bsq_kv4_read(const bsq_kv4_cache_t *cache, const int32_t *d_slots, uint64_t tokens, int type, void *d_k,
                         uint64_t ldk, void *d_v, uint64_t ldv, void *stream);

/* Attention: request r has the keys and values 0 .. d_lengths[r] - 1, in the
 * pages of its row of d_table, and the queries d_starts[r] .. d_starts[r + 1] - 1
 * of `tokens` (d_starts NULL: query r), `most` of them at most; its last query
 * is at the last key's position.  Query head h reads head h / (q_heads / heads)
 * of keys and values:
 *   out = sum over the seen j of softmax(scale q . k[j]) v[j]
 * (|scale| up to 2.35e38).
 * `causal`: a query sees the keys up to its own position, with a `window` above
 * zero only the last `window` of them; else all of its request's (window 0).
 * Keys on page numbers outside the cache are not seen.  A query that sees none
 * gives zeros.  d_lse (tokens x q_heads, may be NULL): the natural logarithm of
 * the softmax's sum, minus infinity where no key is seen.  Sums and softmax are
 * FP32, and so are the scores before their scale: a query whose scores are all
 * below FP32's range gives zeros too.  One that holds an infinity or a NaN gives
 * NaN if it sees a key.  Products with queries are exact to FP32 in every type
 * (FP32 queries in steps of 2^-133), the softmax's weights are rounded to BF16 where
 * both q and out are BF16, are held to 16 bits where FP16 is the finest type among
 * them, and to FP32 where one is FP32.  Queries behind the last request's, and past
 * `most`, are left as they are.  Starts do not fall: of queries that two requests
 * have, the results are either's or left as they are.  The tokens of a request that
 * the plan did not serve lie between its starts like others, and get what they
 * would as the last of the keys that it holds: their results mean nothing.  out
 * may not lie on the queries' rows. */
BSQ_API uint64_t bsq_kv4_attention_workspace(const bsq_kv4_cache_t *cache, uint32_t width, uint32_t requests,
                                             uint64_t tokens, uint32_t most, uint32_t q_heads);
BSQ_API int bsq_kv4_attention(const bsq_kv4_cache_t *cache, const int32_t *d_table, uint32_t width,
                              const int32_t *d_lengths, const int32_t *d_starts, uint32_t requests, const void *d_q,
                              int q_type, uint64_t tokens, uint32_t most, uint32_t q_heads, uint64_t ldq, float scale,
                              int causal, uint32_t window, void *d_out, int out_type, uint64_t ldo, float *d_lse,
                              void *d_work, uint64_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* BITSQZ_LLM_C_H */
