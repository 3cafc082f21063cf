// Products of MX4 matrices on the scaled matrix instructions (mx4.hpp).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes, per lane, one row's block of 32
// codes (16 bytes) of each operand and the two blocks' scale bytes, and sums
// scale_a scale_b (a . b) in FP32.  Lane l holds row l % 32 and block l / 32 of
// two; as the sum over blocks has no order of its own, step s of a slice of
// eight blocks gives lanes 0-31 block s and lanes 32-63 block 4 + s, so a
// lane's four scale bytes of a slice are one aligned word and the instruction
// picks byte s itself.
#include "mx4.hpp"

#include <algorithm>
#include <type_traits>

namespace bsq {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) void glb_void_t;

constexpr int kThreads = 256;
constexpr uint32_t kCodeBytes = kMx4Slice / 2;             // of a row's slice
constexpr uint32_t kScaleBytes = kMx4Slice / kMx4Block;    // of a row's slice

__device__ __forceinline__ void dma16(const uint8_t *g, const uint8_t *l) {
    __builtin_amdgcn_global_load_lds((glb_void_t *)(g), (lds_void_t *)(reinterpret_cast<size_t>(l)), 16, 0, 0);
}
__device__ __forceinline__ void dma4(const uint8_t *g, const uint8_t *l) {
    __builtin_amdgcn_global_load_lds((glb_void_t *)(g), (lds_void_t *)(reinterpret_cast<size_t>(l)), 4, 0, 0);
}

// all LDS operations of this wave and all but its PENDING newest vector
// memory operations are done, then the workgroup barrier
template <int PENDING>
__device__ __forceinline__ void stage_barrier() {
    static_assert(PENDING >= 0 && PENDING < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x070 | (PENDING & 15) | ((PENDING >> 4) << 14));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int STEP>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
    const i32x8 a8 = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]), 0, 0, 0, 0};
    const i32x8 b8 = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, STEP, static_cast<int>(sa), STEP,
                                                           static_cast<int>(sb));
}

enum Mode { kDense, kRows, kShared };

// The tile of BM slots number t of the experts' tiles: the expert (experts
// itself for the slots of none, `experts + 1` past the last tile) and its slots.
struct SlotTile {
    uint32_t expert, begin, end;
};
__device__ __forceinline__ SlotTile slot_tile(const Mx4Product &p, uint32_t pairs, uint32_t t, uint32_t tile) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t e0 = 0; e0 <= p.experts; e0 += 64) {
        const uint32_t e = e0 + lane;
        uint32_t lo = 0, hi = 0;
        if (e <= p.experts) {
            lo = static_cast<uint32_t>(p.offsets[e]);
            hi = e < p.experts ? static_cast<uint32_t>(p.offsets[e + 1]) : pairs;
        }
        const uint32_t n = (hi - lo + tile - 1) / tile;
        uint32_t sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t v = __shfl_up(sum, d);
            sum += lane >= static_cast<uint32_t>(d) ? v : 0u;
        }
        const uint64_t over = __ballot(sum > t);
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            const uint32_t before = __builtin_amdgcn_readlane(sum - n, at);
            const uint32_t begin = __builtin_amdgcn_readlane(lo, at) + (t - before) * tile;
            const uint32_t end = __builtin_amdgcn_readlane(hi, at);
            return {e0 + at, begin, min(begin + tile, end)};
        }
        t -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {p.experts + 1, 0, 0};
}

// T x T tiles, four waves of T/2 x T/2, slices of 256 values: the codes and
// scales of a slice's rows go global -> LDS directly, two slices deep.  A
// row's eight 16-byte blocks are stored in the order block ^ (row % 8), so that
// eight neighbouring rows' reads of one block cover all banks; the permutation
// is made by the lanes' source addresses.
template <int T, Mode MODE, Mx4Type O>
__global__ __launch_bounds__(kThreads) void mx4_product_kernel(Mx4Product p, uint32_t tiles_n, uint32_t pairs) {
    constexpr int B = T / 64;          // 32 x 32 blocks of a wave, each way
    constexpr int kRowLoads = T / 32;  // 16-byte transfers of a lane per operand and slice
    struct Stage {
        uint8_t a[T * kCodeBytes], b[T * kCodeBytes], sa[T * kScaleBytes], sb[T * kScaleBytes];
    };
    // an object each, so that reads of one are not held for transfers to the other
    __shared__ __attribute__((aligned(1024))) Stage s0, s1;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
    uint32_t m0 = tm * T, m_end = p.M, expert = 0, slice0 = 0, slices = p.slices;
    if constexpr (MODE == kRows) {
        const SlotTile s = slot_tile(p, pairs, tm, T);
        if (s.expert > p.experts) return;  // uniform
        expert = s.expert;
        m0 = s.begin;
        m_end = s.end;
        if (expert == p.experts) slices = 0;  // slots of no expert: zero rows
    } else if constexpr (MODE == kShared) {
        expert = blockIdx.y;
        uint32_t before = 0;
        for (uint32_t e = lane; e < expert; e += 64) before += mx4_slot_slices(p.offsets, e);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
        slice0 = __builtin_amdgcn_readfirstlane(before);
        slices = __builtin_amdgcn_readfirstlane(mx4_slot_slices(p.offsets, expert));
    }
    const uint32_t n0 = tn * T;
    const uint32_t b_first = MODE == kRows ? min(expert, p.experts - 1) * p.N : 0u;

    // this lane's rows and blocks of the transfers (rows past the end repeat
    // the last one; their results are not stored)
    const uint8_t *ga[kRowLoads], *gb[kRowLoads];
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) {
        const uint32_t r = 8 * (4 * i + wave) + (lane >> 3), block = (lane & 7) ^ (r & 7);
        uint64_t ra = min(m0 + r, m_end - 1);
        if constexpr (MODE == kRows) ra = static_cast<uint32_t>(p.order[ra]) / p.per_token;
        const uint64_t rb = static_cast<uint64_t>(b_first) + min(n0 + r, p.N - 1);
        ga[i] = p.a.codes + (ra * p.slices + slice0) * kCodeBytes + 16 * block;
        gb[i] = p.b.codes + (rb * p.slices + slice0) * kCodeBytes + 16 * block;
    }
    constexpr int kScaleLoads = T / 128;  // 4-byte transfers of a lane per operand and slice
    const uint8_t *gsa[kScaleLoads], *gsb[kScaleLoads];
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
        const uint32_t r = 32 * (4 * i + wave) + (lane >> 1);
        uint64_t ra = min(m0 + r, m_end - 1);
        if constexpr (MODE == kRows) ra = static_cast<uint32_t>(p.order[ra]) / p.per_token;
        const uint64_t rb = static_cast<uint64_t>(b_first) + min(n0 + r, p.N - 1);
        gsa[i] = p.a.scales + (ra * p.slices + slice0) * kScaleBytes + 4 * (lane & 1);
        gsb[i] = p.b.scales + (rb * p.slices + slice0) * kScaleBytes + 4 * (lane & 1);
    }
    auto fetch = [&](const Stage &s, uint32_t k) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        const uint64_t c = static_cast<uint64_t>(k) * kCodeBytes, f = static_cast<uint64_t>(k) * kScaleBytes;
#pragma unroll
        for (int i = 0; i < kRowLoads; ++i) {
            dma16(ga[i] + c, s.a + 1024 * (4 * i + wave));
            dma16(gb[i] + c, s.b + 1024 * (4 * i + wave));
        }
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i) {
            dma4(gsa[i] + f, s.sa + 256 * (4 * i + wave));
            dma4(gsb[i] + f, s.sb + 256 * (4 * i + wave));
        }
        asm volatile("" ::: "memory");
    };
    constexpr int kLoads = 2 * (kRowLoads + kScaleLoads);

    f32x16 acc[B][B] = {};
    const int wm = (wave >> 1) * (T / 2), wn = (wave & 1) * (T / 2), row = lane & 31, half = lane >> 5;
    auto multiply = [&](const Stage &s) __attribute__((always_inline)) {
        uint32_t sa[B], sb[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            sa[i] = *reinterpret_cast<const uint32_t *>(s.sa + (wm + 32 * i + row) * kScaleBytes + 4 * half);
            sb[i] = *reinterpret_cast<const uint32_t *>(s.sb + (wn + 32 * i + row) * kScaleBytes + 4 * half);
        }
        auto step = [&](auto st) __attribute__((always_inline)) {
            constexpr int S = decltype(st)::value;
            const int unit = 16 * ((4 * half + S) ^ (row & 7));
            u32x4 a[B], b[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                a[i] = *reinterpret_cast<const u32x4 *>(s.a + (wm + 32 * i + row) * kCodeBytes + unit);
                b[i] = *reinterpret_cast<const u32x4 *>(s.b + (wn + 32 * i + row) * kCodeBytes + unit);
            }
#pragma unroll
            for (int i = 0; i < B; ++i)
#pragma unroll
                for (int j = 0; j < B; ++j) acc[i][j] = mfma<S>(a[i], b[j], acc[i][j], sa[i], sb[j]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    };

    auto slice = [&](const Stage &here, const Stage &next, uint32_t k) __attribute__((always_inline)) {
        if (k + 1 < slices) {
            fetch(next, k + 1);
            stage_barrier<kLoads>();
        } else {
            stage_barrier<0>();
        }
        multiply(here);
        stage_barrier<63>();  // its LDS reads are done before the stage is filled again
    };
    if (slices > 0) {
        fetch(s0, 0);
        for (uint32_t k = 0; k < slices; k += 2) {
            slice(s0, s1, k);
            if (k + 1 < slices) slice(s1, s0, k + 1);
        }
    }
    // lane: column n = lane % 32 of a block, rows 8 (q / 4) + 4 (lane / 32) + q % 4
    const uint64_t out0 = MODE == kShared ? static_cast<uint64_t>(expert) * p.M : 0u;
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const uint32_t m = m0 + wm + 32 * i + 8 * (q >> 2) + 4 * half + (q & 3);
            if (m >= m_end) continue;
            uint64_t at = out0 + m;
            if constexpr (MODE == kRows) at = static_cast<uint32_t>(p.order[m]);
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const uint32_t n = n0 + wn + 32 * j + row;
                if (n < p.N) store_value<O>(p.out, at * p.ld + n, acc[i][j][q]);
            }
        }
}

}  // namespace

uint64_t mx4_product_workspace(uint32_t, uint32_t, uint32_t) { return 0; }

void launch_mx4_product(const Mx4Product &p, void *, uint64_t, hipStream_t stream) {
    if (p.M == 0 || p.N == 0) return;
    constexpr uint32_t T = 128;
    const uint64_t tiles_n = ceil_div(p.N, T);
    by_type(p.type, [&](auto t) {
        constexpr Mx4Type O = decltype(t)::value;
        if (p.shared_slots) {
            const uint64_t grid = tiles_n * ceil_div(p.M, T);
            BSQ_REQUIRE(grid <= 0x7FFFFFFFull && p.experts <= 65535, "mx4 product: too large");
            mx4_product_kernel<T, kShared, O><<<dim3(static_cast<unsigned>(grid), p.experts), kThreads, 0, stream>>>(
                p, static_cast<uint32_t>(tiles_n), 0);
        } else if (p.offsets != nullptr) {
            // M: the pairs
            const uint64_t grid = tiles_n * (ceil_div(p.M, T) + p.experts + 1);
            BSQ_REQUIRE(grid <= 0x7FFFFFFFull, "mx4 product: too large");
            mx4_product_kernel<T, kRows, O><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(
                p, static_cast<uint32_t>(tiles_n), p.M);
        } else {
            const uint64_t grid = tiles_n * ceil_div(p.M, T);
            BSQ_REQUIRE(grid <= 0x7FFFFFFFull, "mx4 product: too large");
            mx4_product_kernel<T, kDense, O><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(
                p, static_cast<uint32_t>(tiles_n), 0);
        }
    });
    BSQ_HIP(hipGetLastError());
}

}  // namespace bsq
