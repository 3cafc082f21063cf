// Microscaled 4-bit matrices (MX4): the packed layout and what its kernels
// share (mx4.hip, mx4_gemm.hip, moe.hip).
//
// Blocks of 32 values along a row share a power of two, the smallest 2^e with
// e >= -126 at which no value of the block lies above 6 in magnitude; a value
// over its scale is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties
// to the even code) and its sign (E2M1).  A block that holds a NaN or an
// infinity is NaN as a whole: scale byte 255, codes 0.
//
// A packed matrix of rows x cols: row-major codes, two a byte with the first
// in the low half, and row-major scale bytes (e + 127).  Rows are padded with
// zeros to a multiple of 256 values: 128 bytes of codes (a cache line) and 8 of
// scales, so that no kernel meets a partial slice or an unaligned row.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "bsq_internal.hpp"

namespace bsq {

constexpr uint32_t kMx4Slice = 256;  // values a row is padded to
constexpr uint32_t kMx4Block = 32;

__host__ __device__ inline uint64_t mx4_slices(uint64_t cols) { return (cols + kMx4Slice - 1) / kMx4Slice; }

enum class Mx4Type : int { F32 = 0, BF16 = 1, F16 = 2 };
inline uint32_t type_bytes(Mx4Type t) { return t == Mx4Type::F32 ? 4u : 2u; }

struct Mx4Matrix {
    const uint8_t *codes = nullptr;
    const uint8_t *scales = nullptr;
};

// Where the columns of an encode come from when they are the slots of experts:
// slot s of the order is row order[s] / per_token of x, scaled by
// weights[order[s]] if given; expert e has the slots offsets[e] ..
// offsets[e + 1], padded to whole slices of its own.
struct Mx4Slots {
    const int32_t *offsets = nullptr;
    const int32_t *order = nullptr;
    const float *weights = nullptr;
    uint32_t experts = 0, per_token = 1;
};

// x: `batch` matrices of rows x cols, rows `ld` and matrices `stride` elements
// apart.  rows_out / cols_out (either may be empty): the packed matrices of
// their rows and of their columns (the transposes'), batch after batch.
void launch_mx4_encode(const void *x, Mx4Type type, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t ld,
                       uint64_t stride, uint8_t *codes, uint8_t *scales, uint8_t *codes_t, uint8_t *scales_t,
                       hipStream_t stream);
// Whether the tiles of an encode that writes the columns fit a launch; for calls
// that queue other work before it, and likewise the checks below.
void check_mx4_encode(Mx4Type type, uint64_t batch, uint64_t rows, uint64_t cols);
void launch_mx4_decode(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint64_t cols, void *out,
                       Mx4Type type, uint64_t ld, hipStream_t stream);
// The transpose of the slots' rows (cols x slots, `slices` slices of 256 slots
// a row), every expert's slots from a slice of its own.
void launch_mx4_encode_slots(const void *x, Mx4Type type, uint64_t cols, uint64_t ld, const Mx4Slots &slots,
                             uint64_t slices, uint8_t *codes_t, uint8_t *scales_t, hipStream_t stream);
void check_mx4_encode_slots(Mx4Type type, uint64_t cols, uint64_t slices);

// Both of those for the weighted gradients d (tokens x n) and the inputs x, and
// the rows of d, in one launch; d and x of one type.
void launch_mx4_encode_backward(const void *d, uint64_t n, uint64_t ldd, const void *x, uint64_t inputs, uint64_t ldx,
                                Mx4Type type, uint64_t tokens, Mx4Slots slots, uint64_t slices, uint8_t *dc, uint8_t *ds,
                                uint8_t *xc, uint8_t *xs, uint8_t *rc, uint8_t *rs, hipStream_t stream);
void check_mx4_encode_backward(Mx4Type type, uint64_t n, uint64_t inputs, uint64_t tokens, uint64_t slices);

// Products of packed matrices: out[m, n] = sum over the shared axis.
struct Mx4Product {
    Mx4Matrix a, b;
    uint32_t M = 0, N = 0;      // rows of a and b (of one expert's b)
    uint32_t slices = 0;        // slices of a row of a and b
    void *out = nullptr;
    Mx4Type type = Mx4Type::F32;
    uint64_t ld = 0;
    // rows of a chosen by the experts' order: slot s multiplies row
    // order[s] / per_token of a with expert e's b and writes row order[s]
    const int32_t *offsets = nullptr, *order = nullptr;
    uint32_t experts = 0, per_token = 1;
    // the experts' slots are the shared axis instead: out[e] (M x N) sums the
    // slices of expert e
    bool shared_slots = false;
};
uint64_t mx4_product_workspace(uint32_t M, uint32_t N, uint32_t slices);
void launch_mx4_product(const Mx4Product &p, void *workspace, uint64_t workspace_bytes, hipStream_t stream);
void check_mx4_product(const Mx4Product &p);
// The same with a packed from dense x on the way, for m rows where that pays.
bool mx4_packs_on_the_way(uint64_t m, uint64_t n, uint64_t slices);
void launch_mx4_product_of(const void *x, Mx4Type x_type, uint64_t x_cols, uint64_t ldx, const Mx4Product &p,
                           hipStream_t stream);

// First slice of expert e's slots and the number of slices of all.
__device__ __forceinline__ uint32_t mx4_slot_slices(const int32_t *offsets, uint32_t e) {
    return (static_cast<uint32_t>(offsets[e + 1] - offsets[e]) + kMx4Slice - 1) / kMx4Slice;
}

// The sum of v over the lanes up to this one, by moves within rows of 16 lanes
// and of the rows' last lanes.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    auto moved = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value,
                                                                 decltype(rows)::value, 0xF, false));
    };
    using All = std::integral_constant<int, 0xF>;
    v += moved(std::integral_constant<int, 0x111>{}, All{});
    v += moved(std::integral_constant<int, 0x112>{}, All{});
    v += moved(std::integral_constant<int, 0x114>{}, All{});
    v += moved(std::integral_constant<int, 0x118>{}, All{});
    v += moved(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    v += moved(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return v;
}

// 2^(b - 127), b in [1, 254]
__device__ __forceinline__ float mx4_power(uint32_t b) { return __uint_as_float(b << 23); }

// The scale byte of a block whose largest magnitude has the FP32 bits `top`:
// top / 6 <= 2^e where top / 4 = 1.m 2^e with 1.m <= 1.5, else 2^(e + 1).  NaN
// and infinity: 255.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) {
    const uint32_t b = (top + 0x3FFFFFu) >> 23;
    return top >= 0x7F800000u ? 255u : (b < 3u ? 1u : b - 2u);
}

__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }
// FP32 -> BF16, round to nearest even; NaN stays NaN
__device__ __forceinline__ uint32_t bf16_bits(float f) {
    const uint32_t u = __float_as_uint(f);
    return fabsf(f) <= __builtin_inff() ? (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16 : (u >> 16) | 0x40u;
}
__device__ __forceinline__ uint32_t f16_bits(float f) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(f)));
}
__device__ __forceinline__ float f16_value(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}

template <Mx4Type T>
__device__ __forceinline__ float load_value(const void *p, uint64_t i) {
    if constexpr (T == Mx4Type::F32) return static_cast<const float *>(p)[i];
    const uint32_t b = static_cast<const uint16_t *>(p)[i];
    return T == Mx4Type::BF16 ? bf16_value(b) : f16_value(b);
}
template <Mx4Type T>
__device__ __forceinline__ void store_value(void *p, uint64_t i, float v) {
    if constexpr (T == Mx4Type::F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(T == Mx4Type::BF16 ? bf16_bits(v) : f16_bits(v));
}

typedef _Float16 mx4_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx4_bf16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t mx4_u16x2 __attribute__((ext_vector_type(2)));

// Eight consecutive values in their own type.
template <Mx4Type T>
struct Eight {
    static constexpr int kWords = T == Mx4Type::F32 ? 8 : 4;
    uint32_t w[kWords];

    // values [at, at + 8) of a row of n, zeros past its end; any alignment of
    // the element's own size
    __device__ __forceinline__ void load(const uint8_t *row, uint64_t at, uint64_t n) {
        constexpr int size = T == Mx4Type::F32 ? 4 : 2;
        if (at + 8 <= n) {
            __builtin_memcpy(w, row + at * size, 8 * size);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (at + i >= n) continue;
                if constexpr (T == Mx4Type::F32) w[i] = reinterpret_cast<const uint32_t *>(row)[at + i];
                else w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(row)[at + i]) << (16 * (i & 1));
            }
        }
    }
    // bits of the largest magnitude, in the type's own format (they order as
    // the magnitudes do, infinity and NaN above all)
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (T == Mx4Type::F32) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            mx4_u16x2 m = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(mx4_u16x2, w[i] & 0x7FFF7FFFu));
            return max(static_cast<uint32_t>(m[0]), static_cast<uint32_t>(m[1]));
        }
    }
    // the eight codes over `scale`
    __device__ __forceinline__ uint32_t codes(float scale) const {
        uint32_t c = 0;
        if constexpr (T == Mx4Type::F32) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[0]), __uint_as_float(w[1]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[2]), __uint_as_float(w[3]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[4]), __uint_as_float(w[5]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[6]), __uint_as_float(w[7]), scale, 3);
        } else if constexpr (T == Mx4Type::BF16) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, w[0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, w[1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, w[2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, w[3]), scale, 3);
        } else {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(mx4_f16x2, w[0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(mx4_f16x2, w[1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(mx4_f16x2, w[2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(mx4_f16x2, w[3]), scale, 3);
        }
        return c;
    }
};

// the type's magnitude bits as FP32's
template <Mx4Type T>
__device__ __forceinline__ uint32_t f32_bits(uint32_t top) {
    if constexpr (T == Mx4Type::F32) return top;
    if constexpr (T == Mx4Type::BF16) return top << 16;
    return __float_as_uint(f16_value(top));
}

// Eight consecutive values in FP32
template <Mx4Type T>
__device__ __forceinline__ void load8(const void *base, uint64_t at, uint32_t valid, float v[8]) {
    if (valid >= 8) {
        if constexpr (T == Mx4Type::F32) {
            __builtin_memcpy(v, static_cast<const float *>(base) + at, 32);
        } else {
            uint32_t w[4];
            __builtin_memcpy(w, static_cast<const uint16_t *>(base) + at, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = (w[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
                v[i] = T == Mx4Type::BF16 ? bf16_value(b) : f16_value(b);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<uint32_t>(i) < valid ? load_value<T>(base, at + i) : 0.0f;
    }
}
// Two values rounded to the nearest of a 16-bit type (BF16 in one instruction).
template <Mx4Type T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (T == Mx4Type::BF16) {
        const mx4_bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
        return __builtin_bit_cast(uint32_t, v);
    } else {
        return f16_bits(lo) | (f16_bits(hi) << 16);
    }
}
template <Mx4Type T>
__device__ __forceinline__ void store8(void *base, uint64_t at, uint32_t valid, const float v[8]) {
    if (valid >= 8) {
        if constexpr (T == Mx4Type::F32) {
            __builtin_memcpy(static_cast<float *>(base) + at, v, 32);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
            __builtin_memcpy(static_cast<uint16_t *>(base) + at, w, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (static_cast<uint32_t>(i) < valid) store_value<T>(base, at + i, v[i]);
    }
}

// max over each aligned quad of lanes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
}

// Rows to MX4.  A lane takes eight consecutive values, a quad of lanes a
// block; loads are 16 bytes a lane (twice for FP32), a wave's codes 256
// consecutive bytes.  Workgroup `group` of `groups` of THREADS.
struct Mx4Rows {
    const uint8_t *x;
    uint64_t rows, cols, ld, stride, total;  // total: the batch's rows
    uint32_t chunks;                         // of eight values in a padded row
    uint8_t *codes, *scales;
};
template <Mx4Type T, int THREADS>
__device__ __forceinline__ void encode_rows(const Mx4Rows &r, uint32_t group, uint32_t groups) {
    constexpr int size = T == Mx4Type::F32 ? 4 : 2;
    const uint64_t all = r.total * r.chunks;  // a multiple of 32 a row: quads never part
    for (uint64_t t = static_cast<uint64_t>(group) * THREADS + threadIdx.x; t < all;
         t += static_cast<uint64_t>(groups) * THREADS) {
        const uint64_t row = t / r.chunks, c = t - row * r.chunks, b = row / r.rows;
        Eight<T> v;
        v.load(r.x + (b * r.stride + (row - b * r.rows) * r.ld) * size, 8 * c, r.cols);
        const uint32_t byte = mx4_scale_byte(f32_bits<T>(quad_max(v.top())));
        reinterpret_cast<uint32_t *>(r.codes)[t] = byte == 255u ? 0u : v.codes(mx4_power(byte));
        if ((c & 3) == 0) r.scales[t >> 2] = static_cast<uint8_t>(byte);
    }
}

// fn<T>() for the type of a call
template <class F>
void by_type(Mx4Type t, F &&fn) {
    switch (t) {
        case Mx4Type::F32: fn(std::integral_constant<Mx4Type, Mx4Type::F32>{}); return;
        case Mx4Type::BF16: fn(std::integral_constant<Mx4Type, Mx4Type::BF16>{}); return;
        case Mx4Type::F16: fn(std::integral_constant<Mx4Type, Mx4Type::F16>{}); return;
    }
    fail("mx4: unknown element type");
}

// The grid of a launch.  Its threads are counted in 32 bits: past those the
// runtime cuts the grid without an error.
inline unsigned grid_of(uint64_t groups, uint64_t threads, const char *too_large) {
    BSQ_REQUIRE(groups <= 0xFFFFFFFFull / threads, too_large);
    return static_cast<unsigned>(groups);
}
// The same for kernels whose workgroups go on from item to item.
inline unsigned grid_over(uint64_t groups) { return static_cast<unsigned>(groups < (1u << 20) ? groups : 1u << 20); }

// Checks of a call's arguments.
inline Mx4Type type_of(int t) {
    BSQ_REQUIRE(t >= 0 && t <= 2, "unknown element type");
    return static_cast<Mx4Type>(t);
}
inline void check_packed(const void *codes, const void *scales) {
    BSQ_REQUIRE(codes != nullptr && scales != nullptr, "null packed matrix");
    BSQ_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 15) == 0 && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
                "packed codes are 16-byte and scales 8-byte aligned");
}
inline void check_dense(const void *p, Mx4Type t, const char *null) {
    BSQ_REQUIRE(p != nullptr, null);
    BSQ_REQUIRE((reinterpret_cast<uintptr_t>(p) & (type_bytes(t) - 1)) == 0, "matrix unaligned to its elements");
}
inline void check_work(const void *p, uint64_t bytes, uint64_t need) {
    BSQ_REQUIRE(bytes >= need, "workspace too small");
    if (need > 0) check_packed(p, p);  // begins with codes
}
inline uint64_t round256(uint64_t v) { return (v + 255) & ~255ull; }
inline uint64_t packed_bytes(uint64_t rows, uint64_t slices) { return round256(rows * slices * 128) + round256(rows * slices * 8); }

// C entry points: exceptions become return codes
template <class F>
int entry(F &&f) noexcept {
    try {
        f();
        set_last_error("");
        return 0;
    } catch (const std::exception &e) {
        set_last_error(e.what());
    } catch (...) {
        set_last_error("unknown error");
    }
    return 1;
}

// Size queries: UINT64_MAX where there is no size, with the reason as the last
// error
template <class F>
uint64_t size_query(F &&f) noexcept {
    uint64_t size = UINT64_MAX;
    return entry([&] { size = f(); }) == 0 ? size : UINT64_MAX;
}

}  // namespace bsq
