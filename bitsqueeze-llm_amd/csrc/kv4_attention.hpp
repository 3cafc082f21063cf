// What the attention kernels share (kv4_attention.hip: few queries; kv4_prompt.hip:
// many).
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(x_ij - m_i), x_ij = scale log2(e)
// q_i . k_j, in one pass over the keys with m_i a running reference.  m_i is
// raised only where some x_ij lies more than 8 above it: the sums are FP32, so a
// reference that is up to 2^8 low costs nothing, and most tiles need no rescale
// and no exchange between lanes.
//
// Keys and values are converted to BF16, which holds E2M1 times a power of two
// exactly, and multiplied on the BF16 matrix instructions; queries that BF16 does
// not hold are split into two (FP16) or three (FP32) BF16 pieces, so that products
// are those of FP32.  The weights p go in the same number of pieces.
#pragma once

#include "kv4.hpp"

namespace bsq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t kTileRows = 16;       // rows of a tile of few queries; a row is a (token, head of the group)
constexpr uint32_t kPromptRows = 128;    // and of a prompt's
constexpr int kPromptThreads = 256;
constexpr float kSlack = 8.0f;           // of the reference under the largest score

struct AttentionArgs {
    Kv4Cache cache;
    const int32_t *table, *lengths, *starts;
    uint32_t width, requests;
    const uint8_t *q;
    Mx4Type q_type, out_type;
    uint64_t ldq, ldo;
    uint32_t tokens, most, group;  // group: query heads to a head of keys
    float factor;                  // scale log2(e), not below zero
    bool negate;                   // the scale is below zero
    bool causal;
    uint32_t window;
    uint8_t *out;
    float *lse;
    float *parts;
    struct Split *splits;
    uint32_t few;   // requests of up to so many rows are the one kernel's, others the prompts'
    uint32_t span;  // few queries: a unit of work is 1 << span keys
    uint32_t each;  // prompts: workgroups that share a tile's keys
};

// A tile of queries whose keys more than one workgroup takes: its parts, `rows`
// rows of sums, the reference and their sum (part_row floats, whole 16 bytes), are
// number first, next, next + step ...
struct Split {
    uint32_t parts;  // 0: none
    uint32_t first, next, step;
    uint32_t head, row0, rows, first_token;
};
constexpr uint32_t part_row(uint32_t blocks) { return 32 * blocks + 4; }

struct Request {
    int32_t length, first, count;  // keys, first query, queries
    __device__ __forceinline__ int32_t past() const { return length - count; }
};

__device__ __forceinline__ Request load_request(const AttentionArgs &a, uint32_t r) {
    Request q;
    const int64_t room = static_cast<int64_t>(a.width) << a.cache.shift;
    q.length = static_cast<int32_t>(min(static_cast<int64_t>(max(a.lengths[r], 0)), room));
    if (a.starts == nullptr) {
        q.first = static_cast<int32_t>(r);
        q.count = r < a.tokens ? 1 : 0;
    } else {
        const int32_t tokens = static_cast<int32_t>(a.tokens);
        q.first = min(max(a.starts[r], 0), tokens);
        const int32_t n = min(max(a.starts[r + 1], q.first), tokens) - q.first;
        q.count = min(n, static_cast<int32_t>(a.most));
        // queries past `most` are the last ones: the others' keys end before theirs
        if (a.causal) q.length = max(q.length - (n - q.count), 0);
    }
    return q;
}

// The number of the page of token t, or of the last one's: by a scalar load, which
// is waited for apart from the keys' vector loads.  The table is read only here and
// written by no kernel that runs beside this one.
__device__ __forceinline__ uint32_t page_of(const AttentionArgs &a, uint32_t r, const Request &q, uint32_t t) {
    typedef const __attribute__((address_space(4))) int32_t *Entries;
    const uint32_t last = static_cast<uint32_t>(max(q.length - 1, 0)) >> a.cache.shift;
    return static_cast<uint32_t>(((Entries)(a.table + static_cast<uint64_t>(r) * a.width))[min(t >> a.cache.shift, last)]);
}

__device__ __forceinline__ uint32_t cvt(uint32_t codes, float scale, int byte) {
    switch (byte) {  // an immediate of the instruction
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    }
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Eight FP32 values as P vectors of BF16 whose sums they are (to 8 P bits).  QUERIES:
// of any size, infinities among them.  Those that BF16 would round to infinity (above
// 2^128 - 2^119) are BF16's largest, 2^128 - 2^120, and a rest that the other pieces
// hold.  Infinities are NaN: so is a softmax over their products with any keys, but the
// kernels take scores that are all minus infinity for keys that nobody sees.
template <int P, bool QUERIES = false>
__device__ __forceinline__ void pieces(float x[8], u32x4 out[P]) {
    constexpr float kMost = 0x1.FEp127f;
    if constexpr (QUERIES) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += x[i] - x[i];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w;
            if (QUERIES && P > 1 && p == 0)  // a NaN is one in the rest
                w = pack2<Mx4Type::BF16>(__builtin_amdgcn_fmed3f(x[2 * i], -kMost, kMost), __builtin_amdgcn_fmed3f(x[2 * i + 1], -kMost, kMost));
            else
                w = pack2<Mx4Type::BF16>(x[2 * i], x[2 * i + 1]);
            out[p][i] = w;
            if (p + 1 < P) {
                x[2 * i] -= __uint_as_float(w << 16);
                x[2 * i + 1] -= __uint_as_float(w & 0xFFFF0000u);
            }
        }
    }
}

template <class F>
__device__ __forceinline__ void by_device_type(Mx4Type t, F &&fn) {
    if (t == Mx4Type::BF16) fn(std::integral_constant<Mx4Type, Mx4Type::BF16>{});
    else if (t == Mx4Type::F16) fn(std::integral_constant<Mx4Type, Mx4Type::F16>{});
    else fn(std::integral_constant<Mx4Type, Mx4Type::F32>{});
}

// One row's eight channels of the result, or its logarithm: sums over sum, and
// the reference.
__device__ __forceinline__ void write_row(const AttentionArgs &a, uint64_t token, uint32_t head, uint32_t at, float v[8],
                                          float sum, float top) {
    const bool none = top == -__builtin_inff() && sum == 0.0f;
    const float inverse = none ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none ? 0.0f : v[i] * inverse;
    const uint32_t dim = a.cache.dim;
    if (at < dim)
        by_device_type(a.out_type, [&](auto t) {
            store8<decltype(t)::value>(a.out, token * a.ldo + static_cast<uint64_t>(head) * dim + at, dim - at, v);
        });
    if (at == 0 && a.lse != nullptr)
        a.lse[token * a.cache.heads * a.group + head] = none ? top : (top + __log2f(sum)) * 0.6931471805599453f;
}


// Four values, `valid` of them, rounded to their type.
template <Mx4Type T>
__device__ __forceinline__ void store4(uint8_t *base, uint64_t at, uint32_t valid, const float v[4]) {
    if (valid >= 4) {
        if constexpr (T == Mx4Type::F32) {
            __builtin_memcpy(base + at * 4, v, 16);
        } else {
            const uint32_t w[2] = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            __builtin_memcpy(base + at * 2, w, 8);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < valid) store_value<T>(base, at + i, v[i]);
    }
}

template <class F>
void by_blocks(uint32_t blocks, F &&fn) {
    switch (blocks) {
        case 1: fn(std::integral_constant<int, 1>{}); return;
        case 2: fn(std::integral_constant<int, 2>{}); return;
        case 3: fn(std::integral_constant<int, 3>{}); return;
        case 4: fn(std::integral_constant<int, 4>{}); return;
        case 5: fn(std::integral_constant<int, 5>{}); return;
        case 6: fn(std::integral_constant<int, 6>{}); return;
        case 7: fn(std::integral_constant<int, 7>{}); return;
        case 8: fn(std::integral_constant<int, 8>{}); return;
    }
    fail("kv4: unknown head size");
}

// Few queries: a wave takes kStep keys at once.
constexpr int kFewThreads = 256, kFewWaves = kFewThreads / 64;
constexpr uint32_t kStep = 32;
// A tile's work: units of 1 << a.span keys (at least one, which writes the zeros of
// queries that see none), and kExtra more for what a tile costs beside its keys:
// its queries, reference and first keys wait for one another, and its sums are
// written.  0, 1, 2, 3, 4, 6, 8 of them: 145, 108, 92, 81, 77, 77, 78 us for 128
// requests of 16 to 16384 keys, 8 heads of 128; 110.5 to 109 us for 8 of 40 to 90
// thousand, where they hardly count.
constexpr uint32_t kExtra = 4;
// Units that a share has at least: more shares are more parts to join, fewer leave
// waves idle (2, 4, 6, 8, 12: 17.1, 15.8, 17.4, 19.1, 22.3 us for 16 requests of 400
// to 1200 keys, 18.9, 19.5, 18.5, 20.1, 24.5 for 9 of 100 to 5000 in FP32).
constexpr uint32_t kLeast = 4;

// Requests of up to a.few rows, P BF16 pieces, in shares of `waves` waves.
template <int P>
void launch_kv4_few(const AttentionArgs &a, uint32_t waves, hipStream_t stream);

// Requests of more than a.few rows; depth: BF16 pieces.  grid: `tiles` tiles of
// kPromptRows rows (no fewer than there are) times the heads times a.each.  With
// a.each > 1 the parts and splits are tile-major, of each tile and head.
void launch_kv4_prompt(const AttentionArgs &a, int depth, uint64_t tiles, hipStream_t stream);

}  // namespace bsq
