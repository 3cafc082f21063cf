// MX4 encode and decode (mx4.hpp).
#include "mx4.hpp"

#include <algorithm>
#include <type_traits>

#include <bitsqz_llm_c.h>

namespace bsq {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

// Rows to MX4, eight values a lane (encode_rows).  HBM bound where it is large:
// 4096 x 4096 BF16 (43 MB, 8.2 us at the rate of a large copy) 10.4 us; 16 x
// 4096 2.9 us, a launch.
template <Mx4Type T>
__global__ __launch_bounds__(kThreads) void mx4_encode_rows_kernel(Mx4Rows r) {
    encode_rows<T, kThreads>(r, blockIdx.x, gridDim.x);
}

// Columns to MX4, and the rows too if asked.  A workgroup takes a tile of 256
// rows and 64 words of each: 16 lanes load a row's part (and encode its blocks
// from registers), the tile goes to LDS, and a lane then takes one block of 32
// rows of a word's column (two columns of a 16-bit type); the eight lanes of a
// column's eight blocks are neighbours, so that their codes are a whole line.
// Row r of the tile lies 8 words further along for each block of 32 rows
// before it: eight columns of eight blocks then read all 64 banks.  Tiles that
// write the halves of a line of row codes run on one XCD.
// SLOTS: the rows are those of the experts' slots.  WEIGHTED: each times its
// weight, in FP32 as its block is encoded, so that a value is rounded once.
// HBM bound: 4096 x 11008 BF16 both ways, 32 us with x in the last cache, 45
// from HBM among other writes (read once, two packed matrices written: 27 us at
// the rate of a large copy); 16 matrices of 2752 x 2048 64 (53).
constexpr int kTileRows = 256;
constexpr int kTileWords = 64;
constexpr int kTileThreads = 512;
constexpr int kPad = 8, kPasses = kTileRows / 32;
constexpr int kTileWeights = kTileRows * kTileWords + 8 * kPad;  // where the rows' weights lie
constexpr int kTileLds = kTileWeights + kTileRows;

template <Mx4Type T>
constexpr int kTileCols = T == Mx4Type::F32 ? 64 : 128;

struct EncodeTiles {
    const uint8_t *x;
    uint64_t rows, cols, ld, stride;
    uint32_t tiles_c, tiles_r, slices_c, slices_r;
    Mx4Slots slots;
    uint8_t *codes, *scales, *codes_t, *scales_t;
};

// Tile number `group` of `groups`.
template <Mx4Type T, bool SLOTS, bool WEIGHTED>
__device__ __forceinline__ void encode_tile(const EncodeTiles &job, uint32_t *tile, uint32_t group, uint32_t groups) {
    const auto [x, rows, cols, ld, stride, tiles_c, tiles_r, slices_c, slices_r, slots, codes, scales, codes_t, scales_t] = job;
    constexpr int size = T == Mx4Type::F32 ? 4 : 2, kCols = kTileCols<T>, kPer = kCols / 16;
    const int tid = threadIdx.x;
    // each XCD a contiguous run of the tiles
    const uint32_t xcd = group % 8, per = groups / 8, extra = groups % 8;
    const uint32_t number = xcd * per + min(xcd, extra) + group / 8;
    const uint32_t tc = number % tiles_c;
    const uint64_t rest = number / tiles_c;
    const uint32_t tr = static_cast<uint32_t>(rest % tiles_r);
    const uint64_t b = rest / tiles_r;
    const uint64_t c0 = static_cast<uint64_t>(tc) * kCols;
    uint64_t r0 = static_cast<uint64_t>(tr) * kTileRows, r1 = rows;  // rows of the tile end at r1
    if constexpr (SLOTS) {
        // tile tr of the experts' slices: the expert it belongs to, 64 at a time
        const uint32_t lane = tid & 63;
        uint32_t before = 0;
        r1 = 0;
        for (uint32_t e0 = 0; e0 < slots.experts; e0 += 64) {
            const uint32_t e = min(e0 + lane, slots.experts - 1);
            const uint32_t lo = static_cast<uint32_t>(slots.offsets[e]), hi = static_cast<uint32_t>(slots.offsets[e + 1]);
            const uint32_t n = e0 + lane < slots.experts ? (hi - lo + kMx4Slice - 1) / kMx4Slice : 0u;
            const uint32_t sum = wave_prefix(n);
            const uint64_t over = __ballot(before + sum > tr);
            if (over != 0) {
                const int at = __builtin_ctzll(over);
                r0 = __builtin_amdgcn_readlane(lo, at) +
                     (tr - before - __builtin_amdgcn_readlane(sum - n, at)) * static_cast<uint64_t>(kTileRows);
                r1 = __builtin_amdgcn_readlane(hi, at);
                break;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        if (r1 == 0) return;  // uniform: past the last expert's slices
    }
    const int part = tid & 15;
    const uint64_t c = c0 + part * kPer;
    constexpr int kWords = kPer * size / 4;
    uint32_t v[kPasses][kWords];
    float w[kPasses];
    const uint8_t *from[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const uint64_t row = min(r0 + 32 * i + (tid >> 4), r1 - 1);  // past the end: the last row, not used
        from[i] = x + b * stride * size;
        w[i] = 1.0f;
        if constexpr (SLOTS) {
            const uint32_t pair = static_cast<uint32_t>(slots.order[row]);
            from[i] += static_cast<uint64_t>(pair / slots.per_token) * ld * size;
            if constexpr (WEIGHTED) w[i] = slots.weights[pair];
        } else {
            from[i] += row * ld * size;
        }
    }
    if (c + kPer <= cols) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) __builtin_memcpy(v[i], from[i] + c * size, sizeof v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
#pragma unroll
            for (int k = 0; k < kWords; ++k) v[i][k] = 0;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if (c + k >= cols) continue;
                if constexpr (T == Mx4Type::F32) v[i][k] = reinterpret_cast<const uint32_t *>(from[i])[c + k];
                else v[i][k / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(from[i])[c + k]) << (16 * (k & 1));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int r = 32 * i + (tid >> 4);
        const uint64_t row = r0 + r;
#pragma unroll
        for (int k = 0; k < kWords; ++k) v[i][k] = row < r1 ? v[i][k] : 0u;
        u32x4 staged;
#pragma unroll
        for (int k = 0; k < 4; ++k) staged[k] = v[i][k];
        if (WEIGHTED && part == 0) tile[kTileWeights + r] = row < r1 ? __float_as_uint(w[i]) : 0u;
        if (!SLOTS && codes != nullptr) {  // uniform
            uint32_t byte, q = 0;
            if constexpr (T == Mx4Type::F32) {
                uint32_t m = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) m = max(m, v[i][k] & 0x7FFFFFFFu);
                m = quad_max(m);
                m = max(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0x141, 0xF, 0xF, true)));
                byte = mx4_scale_byte(m);
                if (byte != 255u) {
                    const float s = mx4_power(byte);
                    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(v[i][0]), __uint_as_float(v[i][1]), s, 0);
                    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(v[i][2]), __uint_as_float(v[i][3]), s, 1);
                }
            } else {
                Eight<T> e8;
                __builtin_memcpy(e8.w, v[i], 16);
                byte = mx4_scale_byte(f32_bits<T>(quad_max(e8.top())));
                if (byte != 255u) q = e8.codes(mx4_power(byte));
            }
            if (row < rows) {
                const uint64_t at = (b * rows + row) * slices_c * kMx4Slice + c;  // padded element
                if constexpr (T == Mx4Type::F32) reinterpret_cast<uint16_t *>(codes)[at >> 2] = static_cast<uint16_t>(q);
                else reinterpret_cast<uint32_t *>(codes)[at >> 3] = q;
                if ((part & (32 / kPer - 1)) == 0) scales[at >> 5] = static_cast<uint8_t>(byte);
            }
        }
        *reinterpret_cast<u32x4 *>(&tile[r * kTileWords + i * kPad + 4 * part]) = staged;
    }
    __syncthreads();
    const int word = tid >> 3, blk = tid & 7;  // eight lanes: the eight blocks of a word's column
    const uint32_t *p = &tile[blk * (32 * kTileWords + kPad) + word];
    uint32_t u[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i] = p[i * kTileWords];
    float by[32];
    if constexpr (WEIGHTED) __builtin_memcpy(by, &tile[kTileWeights + 32 * blk], sizeof by);
    constexpr int kSub = kCols / kTileWords;  // columns in a word
#pragma unroll
    for (int h = 0; h < kSub; ++h) {
        auto val = [&](int i) __attribute__((always_inline)) {
            float f;
            if constexpr (T == Mx4Type::F32) f = __uint_as_float(u[i]);
            else if constexpr (T == Mx4Type::BF16) f = __uint_as_float(h ? u[i] & 0xFFFF0000u : u[i] << 16);
            else f = f16_value(h ? u[i] >> 16 : u[i] & 0xFFFFu);
            return WEIGHTED ? f * by[i] : f;
        };
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (T == Mx4Type::F32 || WEIGHTED) m = max(m, __float_as_uint(val(i)) & 0x7FFFFFFFu);
            else m = max(m, (h ? u[i] >> 16 : u[i]) & 0x7FFFu);
        }
        const uint32_t byte = mx4_scale_byte(WEIGHTED ? m : f32_bits<T>(m));
        const float s = mx4_power(byte);
        u32x4 q = {0, 0, 0, 0};
        if (byte != 255u) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t o = 0;
                o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, val(8 * k), val(8 * k + 1), s, 0);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, val(8 * k + 2), val(8 * k + 3), s, 1);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, val(8 * k + 4), val(8 * k + 5), s, 2);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, val(8 * k + 6), val(8 * k + 7), s, 3);
                q[k] = o;
            }
        }
        const uint64_t col = c0 + static_cast<uint64_t>(word) * kSub + h;
        if (col < cols) {
            const uint64_t at = (b * cols + col) * slices_r + tr;  // slices before this one
            *reinterpret_cast<u32x4 *>(codes_t + at * 128 + blk * 16) = q;
            scales_t[at * 8 + blk] = static_cast<uint8_t>(byte);
        }
    }
}

template <Mx4Type T, bool SLOTS, bool WEIGHTED>
__global__ __launch_bounds__(kTileThreads) void mx4_encode_tile_kernel(EncodeTiles job) {
    __shared__ __attribute__((aligned(16))) uint32_t tile[kTileLds];
    encode_tile<T, SLOTS, WEIGHTED>(job, tile, blockIdx.x, gridDim.x);
}

// What the gradients of the experts' layer multiply, in one launch: the
// weighted gradients' and the inputs' columns by experts, and the gradients'
// rows.  None needs another; three launches took 8 us more.  2048 tokens of
// two pairs each, 2752 and 2048 BF16: 24 us for 75 MB, mostly from the caches:
// the chain of a tile's loads (its expert, its pairs, their rows) bounds it.
template <Mx4Type T>
__global__ __launch_bounds__(kTileThreads) void mx4_encode_backward_kernel(EncodeTiles d, uint32_t d_groups, EncodeTiles x,
                                                                           uint32_t x_groups, Mx4Rows rows) {
    __shared__ __attribute__((aligned(16))) uint32_t tile[kTileLds];
    const uint32_t g = blockIdx.x;
    if (g < d_groups) encode_tile<T, true, true>(d, tile, g, d_groups);
    else if (g < d_groups + x_groups) encode_tile<T, true, false>(x, tile, g - d_groups, x_groups);
    else encode_rows<T, kTileThreads>(rows, g - d_groups - x_groups, gridDim.x - d_groups - x_groups);
}

// Values of packed rows.  A lane takes eight codes; the level of a code times
// its power of two is exact in FP32 and in BF16, and in FP16 rounded once where
// it leaves that type's range.  HBM bound: 4096 x 11008 to BF16 22 us (114 MB,
// the rate of a large copy).
template <Mx4Type T>
__global__ __launch_bounds__(kThreads) void mx4_decode_kernel(const uint8_t *__restrict__ codes,
                                                              const uint8_t *__restrict__ scales, uint64_t rows,
                                                              uint64_t cols, uint64_t slices, uint32_t chunks,
                                                              uint8_t *__restrict__ out, uint64_t ld) {
    constexpr int size = T == Mx4Type::F32 ? 4 : 2;
    const uint64_t all = rows * chunks;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x; t < all;
         t += static_cast<uint64_t>(gridDim.x) * kThreads) {
        const uint64_t r = t / chunks, c = t - r * chunks;
        const uint32_t q = *reinterpret_cast<const uint32_t *>(codes + r * slices * 128 + 4 * c);
        const uint32_t byte = scales[r * slices * 8 + (c >> 2)];
        const float s = byte == 0u ? 0x1p-127f : mx4_power(byte);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // E2M1 read as the top of an E8M23 word: the exponent counts from
            // 2^-126 there, the subnormal half among them
            const uint32_t k = q >> (4 * i);
            const float level = __uint_as_float(((k & 8u) << 28) | ((k & 7u) << 22)) * 0x1p126f;
            v[i] = byte == 255u ? __builtin_nanf("") : level * s;
        }
        const uint64_t e = 8 * c;
        uint8_t *p = out + (r * ld + e) * size;
        if (e + 8 <= cols) {
            uint32_t w[T == Mx4Type::F32 ? 8 : 4];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                if constexpr (T == Mx4Type::F32) {
                    w[i] = __float_as_uint(v[i]);
                    w[i + 1] = __float_as_uint(v[i + 1]);
                } else if constexpr (T == Mx4Type::BF16) {
                    w[i / 2] = (__float_as_uint(v[i]) >> 16) | (__float_as_uint(v[i + 1]) & 0xFFFF0000u);
                } else {
                    w[i / 2] = f16_bits(v[i]) | (f16_bits(v[i + 1]) << 16);
                }
            }
            __builtin_memcpy(p, w, 8 * size);
        } else {
            for (int i = 0; i < 8; ++i)
                if (e + i < cols) store_value<T>(out, r * ld + e + i, v[i]);
        }
    }
}

unsigned grid_for(uint64_t items) { return grid_over(ceil_div(items, kThreads)); }

constexpr const char *kTooLarge = "mx4 encode: matrix too large";
uint64_t tile_cols(Mx4Type type) { return type == Mx4Type::F32 ? kTileCols<Mx4Type::F32> : kTileCols<Mx4Type::BF16>; }
// whole slices both ways, so that the padding is written too
uint64_t encode_tiles(Mx4Type type, uint64_t batch, uint64_t rows, uint64_t cols) {
    return batch * mx4_slices(cols) * (kMx4Slice / tile_cols(type)) * mx4_slices(rows);
}
uint64_t slot_groups(Mx4Type type, uint64_t cols, uint64_t slices) { return slices * ceil_div(cols, tile_cols(type)); }
uint64_t row_groups(uint64_t tokens, uint64_t n) {
    return grid_over(ceil_div(tokens * mx4_slices(n) * (kMx4Slice / 8), kTileThreads));
}

}  // namespace

void check_mx4_encode(Mx4Type type, uint64_t batch, uint64_t rows, uint64_t cols) {
    grid_of(encode_tiles(type, batch, rows, cols), kTileThreads, kTooLarge);
}
void check_mx4_encode_slots(Mx4Type type, uint64_t cols, uint64_t slices) {
    grid_of(slot_groups(type, cols, slices), kTileThreads, kTooLarge);
}
void check_mx4_encode_backward(Mx4Type type, uint64_t n, uint64_t inputs, uint64_t tokens, uint64_t slices) {
    grid_of(slot_groups(type, n, slices) + slot_groups(type, inputs, slices) + row_groups(tokens, n), kTileThreads, kTooLarge);
}

void launch_mx4_encode(const void *x, Mx4Type type, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t ld,
                       uint64_t stride, uint8_t *codes, uint8_t *scales, uint8_t *codes_t, uint8_t *scales_t,
                       hipStream_t stream) {
    if (batch == 0 || rows == 0 || cols == 0 || (codes == nullptr && codes_t == nullptr)) return;
    const uint32_t slices_c = static_cast<uint32_t>(mx4_slices(cols)), slices_r = static_cast<uint32_t>(mx4_slices(rows));
    by_type(type, [&](auto t) {
        constexpr Mx4Type T = decltype(t)::value;
        const uint8_t *p = static_cast<const uint8_t *>(x);
        if (codes_t == nullptr) {
            const uint32_t chunks = slices_c * (kMx4Slice / 8);
            mx4_encode_rows_kernel<T><<<grid_for(batch * rows * chunks), kThreads, 0, stream>>>(
                Mx4Rows{p, rows, cols, ld, stride, batch * rows, chunks, codes, scales});
        } else {
            constexpr uint32_t kCols = kTileCols<T>;
            const unsigned grid = grid_of(encode_tiles(type, batch, rows, cols), kTileThreads, kTooLarge);
            mx4_encode_tile_kernel<T, false, false><<<grid, kTileThreads, 0, stream>>>(
                EncodeTiles{p, rows, cols, ld, stride, slices_c * (kMx4Slice / kCols), slices_r, slices_c, slices_r,
                            Mx4Slots{}, codes, scales, codes_t, scales_t});
        }
    });
    BSQ_HIP(hipGetLastError());
}

namespace {

template <Mx4Type T>
EncodeTiles slot_tiles(const void *x, uint64_t cols, uint64_t ld, const Mx4Slots &slots, uint64_t slices, uint8_t *codes_t,
                       uint8_t *scales_t) {
    const uint32_t tiles_c = static_cast<uint32_t>(ceil_div(cols, kTileCols<T>));
    return {static_cast<const uint8_t *>(x), 0, cols, ld, 0, tiles_c, static_cast<uint32_t>(slices), 0,
            static_cast<uint32_t>(slices), slots, nullptr, nullptr, codes_t, scales_t};
}

}  // namespace

void launch_mx4_encode_slots(const void *x, Mx4Type type, uint64_t cols, uint64_t ld, const Mx4Slots &slots,
                             uint64_t slices, uint8_t *codes_t, uint8_t *scales_t, hipStream_t stream) {
    if (slices == 0 || cols == 0) return;
    by_type(type, [&](auto t) {
        constexpr Mx4Type T = decltype(t)::value;
        auto go = [&](auto weighted) {
            constexpr bool W = decltype(weighted)::value;
            const unsigned grid = grid_of(slot_groups(type, cols, slices), kTileThreads, kTooLarge);
            mx4_encode_tile_kernel<T, true, W><<<grid, kTileThreads, 0, stream>>>(
                slot_tiles<T>(x, cols, ld, slots, slices, codes_t, scales_t));
        };
        if (slots.weights != nullptr) go(std::true_type{});
        else go(std::false_type{});
    });
    BSQ_HIP(hipGetLastError());
}

void launch_mx4_encode_backward(const void *d, uint64_t n, uint64_t ldd, const void *x, uint64_t inputs, uint64_t ldx,
                                Mx4Type type, uint64_t tokens, Mx4Slots slots, uint64_t slices, uint8_t *dc, uint8_t *ds,
                                uint8_t *xc, uint8_t *xs, uint8_t *rc, uint8_t *rs, hipStream_t stream) {
    by_type(type, [&](auto t) {
        constexpr Mx4Type T = decltype(t)::value;
        const uint64_t d_groups = slot_groups(type, n, slices), x_groups = slot_groups(type, inputs, slices);
        const EncodeTiles of_d = slot_tiles<T>(d, n, ldd, slots, slices, dc, ds);
        slots.weights = nullptr;
        const EncodeTiles of_x = slot_tiles<T>(x, inputs, ldx, slots, slices, xc, xs);
        const Mx4Rows rows{static_cast<const uint8_t *>(d), tokens, n, ldd, 0, tokens,
                           static_cast<uint32_t>(mx4_slices(n)) * (kMx4Slice / 8), rc, rs};
        const unsigned grid = grid_of(d_groups + x_groups + row_groups(tokens, n), kTileThreads, kTooLarge);
        mx4_encode_backward_kernel<T><<<grid, kTileThreads, 0, stream>>>(
            of_d, static_cast<uint32_t>(d_groups), of_x, static_cast<uint32_t>(x_groups), rows);
    });
    BSQ_HIP(hipGetLastError());
}

void launch_mx4_decode(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint64_t cols, void *out,
                       Mx4Type type, uint64_t ld, hipStream_t stream) {
    if (rows == 0 || cols == 0) return;
    by_type(type, [&](auto t) {
        constexpr Mx4Type T = decltype(t)::value;
        const uint32_t chunks = static_cast<uint32_t>(ceil_div(cols, 8));
        mx4_decode_kernel<T><<<grid_for(rows * chunks), kThreads, 0, stream>>>(
            codes, scales, rows, cols, mx4_slices(cols), chunks, static_cast<uint8_t *>(out), ld);
    });
    BSQ_HIP(hipGetLastError());
}

}  // namespace bsq

using namespace bsq;

namespace {

constexpr uint64_t kMaxSide = 1ull << 31;
void check_sides(uint64_t m, uint64_t n, uint64_t k) {
    BSQ_REQUIRE(m < kMaxSide && n < kMaxSide && k <= (1u << 22), "mx4: up to 2^31 rows, 2^22 values a row");
}
uint64_t packed(uint64_t rows, uint64_t cols) { return packed_bytes(rows, mx4_slices(cols)); }

// Workspaces of sizes that are checked; they ask the device for its CUs.
uint64_t product_work(uint64_t m, uint64_t n, uint64_t k) {
    return mx4_product_workspace(static_cast<uint32_t>(m), static_cast<uint32_t>(n), static_cast<uint32_t>(mx4_slices(k)));
}
uint64_t linear_work(uint64_t m, uint64_t n, uint64_t k) { return packed(m, k) + round256(product_work(m, n, k)); }
uint64_t linear_backward_work(uint64_t m, uint64_t n, uint64_t k) {
    return packed(m, n) + packed(n, m) + round256(std::max(product_work(m, k, n), product_work(n, k, m)));
}

Mx4Product product_of(Mx4Matrix a, uint64_t m, Mx4Matrix b, uint64_t n, uint64_t k, void *out, Mx4Type type, uint64_t ld) {
    Mx4Product p;
    p.a = a;
    p.b = b;
    p.M = static_cast<uint32_t>(m);
    p.N = static_cast<uint32_t>(n);
    p.slices = static_cast<uint32_t>(mx4_slices(k));
    p.out = out;
    p.type = type;
    p.ld = ld;
    return p;
}

}  // namespace

extern "C" {

uint64_t bsq_mx4_codes_bytes(uint64_t rows, uint64_t cols) { return rows * mx4_slices(cols) * 128; }
uint64_t bsq_mx4_scales_bytes(uint64_t rows, uint64_t cols) { return rows * mx4_slices(cols) * 8; }

int bsq_mx4_encode(const void *d_x, int type, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t stride,
                   uint8_t *d_codes, uint8_t *d_scales, uint8_t *d_codes_t, uint8_t *d_scales_t, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        check_sides(rows, cols, std::max<uint64_t>(cols, d_codes_t ? rows : 0));
        BSQ_REQUIRE(batch < kMaxSide, "mx4 encode: batch too large");
        BSQ_REQUIRE(ld >= cols, "mx4 encode: rows overlap");
        if (batch == 0 || rows == 0 || cols == 0) return;
        check_dense(d_x, t, "mx4 encode: null input");
        BSQ_REQUIRE(d_codes != nullptr || d_codes_t != nullptr, "mx4 encode: null output");
        BSQ_REQUIRE((d_codes == nullptr) == (d_scales == nullptr) && (d_codes_t == nullptr) == (d_scales_t == nullptr),
                    "mx4 encode: codes come with their scales");
        if (d_codes) check_packed(d_codes, d_scales);
        if (d_codes_t) check_packed(d_codes_t, d_scales_t);
        launch_mx4_encode(d_x, t, batch, rows, cols, ld, stride, d_codes, d_scales, d_codes_t, d_scales_t,
                          static_cast<hipStream_t>(stream));
    });
}

int bsq_mx4_decode(const uint8_t *d_codes, const uint8_t *d_scales, uint64_t rows, uint64_t cols, void *d_out, int type,
                   uint64_t ld, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        check_sides(rows, cols, cols);
        BSQ_REQUIRE(ld >= cols, "mx4 decode: rows overlap");
        if (rows == 0 || cols == 0) return;
        check_packed(d_codes, d_scales);
        check_dense(d_out, t, "mx4 decode: null output");
        launch_mx4_decode(d_codes, d_scales, rows, cols, d_out, t, ld, static_cast<hipStream_t>(stream));
    });
}

uint64_t bsq_mx4_product_workspace(uint64_t m, uint64_t n, uint64_t k) {
    return size_query([&] {
        check_sides(m, n, k);
        return product_work(m, n, k);
    });
}

int bsq_mx4_product(const uint8_t *d_a_codes, const uint8_t *d_a_scales, uint64_t m, const uint8_t *d_b_codes,
                    const uint8_t *d_b_scales, uint64_t n, uint64_t k, void *d_out, int type, uint64_t ld, void *d_work,
                    uint64_t work_bytes, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        check_sides(m, n, k);
        BSQ_REQUIRE(k >= 1, "mx4 product: no values to sum");
        BSQ_REQUIRE(ld >= n, "mx4 product: rows overlap");
        if (m == 0 || n == 0) return;
        check_packed(d_a_codes, d_a_scales);
        check_packed(d_b_codes, d_b_scales);
        check_dense(d_out, t, "mx4 product: null output");
        check_work(d_work, work_bytes, product_work(m, n, k));
        launch_mx4_product(product_of({d_a_codes, d_a_scales}, m, {d_b_codes, d_b_scales}, n, k, d_out, t, ld), d_work,
                           work_bytes, static_cast<hipStream_t>(stream));
    });
}

uint64_t bsq_mx4_linear_workspace(uint64_t m, uint64_t n, uint64_t k) {
    return size_query([&] {
        check_sides(m, n, k);
        return linear_work(m, n, k);
    });
}

int bsq_mx4_linear(const void *d_x, int x_type, uint64_t m, uint64_t k, uint64_t ldx, const uint8_t *d_w_codes,
                   const uint8_t *d_w_scales, uint64_t n, void *d_out, int out_type, uint64_t ldo, uint8_t *d_xt_codes,
                   uint8_t *d_xt_scales, void *d_work, uint64_t work_bytes, void *stream) {
    return entry([&] {
        const Mx4Type tx = type_of(x_type), to = type_of(out_type);
        check_sides(m, n, std::max<uint64_t>(k, d_xt_codes ? m : 0));
        BSQ_REQUIRE(k >= 1, "mx4 linear: no inputs");
        BSQ_REQUIRE(ldx >= k && ldo >= n, "mx4 linear: rows overlap");
        if (m == 0 || n == 0) return;
        check_dense(d_x, tx, "mx4 linear: null input");
        check_dense(d_out, to, "mx4 linear: null output");
        check_packed(d_w_codes, d_w_scales);
        BSQ_REQUIRE((d_xt_codes == nullptr) == (d_xt_scales == nullptr), "mx4 linear: codes come with their scales");
        if (d_xt_codes) check_packed(d_xt_codes, d_xt_scales);
        check_work(d_work, work_bytes, linear_work(m, n, k));
        hipStream_t s = static_cast<hipStream_t>(stream);
        uint8_t *codes = static_cast<uint8_t *>(d_work), *scales = codes + round256(m * mx4_slices(k) * 128);
        const Mx4Product p = product_of({codes, scales}, m, {d_w_codes, d_w_scales}, n, k, d_out, to, ldo);
        if (mx4_packs_on_the_way(m, n, p.slices) && d_xt_codes == nullptr) {
            launch_mx4_product_of(d_x, tx, k, ldx, p, s);
            return;
        }
        if (d_xt_codes != nullptr) check_mx4_encode(tx, 1, m, k);
        check_mx4_product(p);
        launch_mx4_encode(d_x, tx, 1, m, k, ldx, 0, codes, scales, d_xt_codes, d_xt_scales, s);
        launch_mx4_product(p, codes + packed(m, k), work_bytes - packed(m, k), s);
    });
}

uint64_t bsq_mx4_linear_backward_workspace(uint64_t m, uint64_t n, uint64_t k) {
    return size_query([&] {
        check_sides(m, n, std::max({m, n, k}));
        return linear_backward_work(m, n, k);
    });
}

int bsq_mx4_linear_backward(const void *d_dy, int type, uint64_t m, uint64_t n, uint64_t ldy, const uint8_t *d_xt_codes,
                            const uint8_t *d_xt_scales, const uint8_t *d_wt_codes, const uint8_t *d_wt_scales, uint64_t k,
                            void *d_dx, uint64_t lddx, void *d_dw, uint64_t lddw, int g_type, void *d_work,
                            uint64_t work_bytes, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type), tg = type_of(g_type);
        check_sides(m, n, std::max({m, n, k}));
        BSQ_REQUIRE(m >= 1 && n >= 1, "mx4 linear backward: empty");
        BSQ_REQUIRE(ldy >= n && (d_dx == nullptr || lddx >= k) && (d_dw == nullptr || lddw >= k), "mx4 linear backward: rows overlap");
        if (k == 0 || (d_dx == nullptr && d_dw == nullptr)) return;
        check_dense(d_dy, t, "mx4 linear backward: null gradient");
        if (d_dx) check_dense(d_dx, tg, "");
        if (d_dw) check_dense(d_dw, tg, "");
        if (d_dx) check_packed(d_wt_codes, d_wt_scales);
        if (d_dw) check_packed(d_xt_codes, d_xt_scales);
        check_work(d_work, work_bytes, linear_backward_work(m, n, k));
        hipStream_t s = static_cast<hipStream_t>(stream);
        uint8_t *rc = static_cast<uint8_t *>(d_work), *rs = rc + round256(m * mx4_slices(n) * 128);
        uint8_t *cc = rc + packed(m, n), *cs = cc + round256(n * mx4_slices(m) * 128);
        uint8_t *rest = cc + packed(n, m);
        const uint64_t rest_bytes = work_bytes - packed(m, n) - packed(n, m);
        const Mx4Product dx = product_of({rc, rs}, m, {d_wt_codes, d_wt_scales}, k, n, d_dx, tg, lddx);
        const Mx4Product dw = product_of({cc, cs}, n, {d_xt_codes, d_xt_scales}, k, m, d_dw, tg, lddw);
        if (d_dw) check_mx4_encode(t, 1, m, n);
        if (d_dx) check_mx4_product(dx);
        if (d_dw) check_mx4_product(dw);
        launch_mx4_encode(d_dy, t, 1, m, n, ldy, 0, d_dx ? rc : nullptr, d_dx ? rs : nullptr, d_dw ? cc : nullptr,
                          d_dw ? cs : nullptr, s);
        if (d_dx) launch_mx4_product(dx, rest, rest_bytes, s);
        if (d_dw) launch_mx4_product(dw, rest, rest_bytes, s);
    });
}

}  // extern "C"
