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
#include "tile_map.hpp"

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

// A uniform address that stays in scalar registers: added to the lanes' offsets
// ahead of a loop it would take two vector registers for each of them.
template <int G>
__device__ __forceinline__ const uint8_t *scalar(const uint8_t *p) {
    if constexpr (G == 1) asm volatile("" : "+s"(p));  // teams differ within a workgroup
    return p;
}

enum Mode { kDense, kRows, kShared };

// The slots of 64 experts from e0 on, one a lane (`experts` itself: the slots of
// none), and their tiles of `tile` slots: how many, and up to this lane.
struct SlotScan {
    uint32_t begin, end, tiles, sum;
};
__device__ __forceinline__ SlotScan scan_slots(const Mx4Product &p, uint32_t pairs, uint32_t e0, uint32_t tile) {
    const uint32_t e = e0 + (threadIdx.x & 63);
    SlotScan s{0, 0, 0, 0};
    if (e <= p.experts) {
        s.begin = static_cast<uint32_t>(p.offsets[e]);
        s.end = e < p.experts ? static_cast<uint32_t>(p.offsets[e + 1]) : pairs;
    }
    s.tiles = (s.end - s.begin + tile - 1) / tile;
    s.sum = wave_prefix(s.tiles);
    return s;
}
// `first`: the scan of the first 64 experts, which is all of it for most layers.
__device__ __forceinline__ uint32_t slot_tiles(const Mx4Product &p, uint32_t pairs, uint32_t tile, const SlotScan &first) {
    uint32_t count = __builtin_amdgcn_readlane(first.sum, 63);
    for (uint32_t e0 = 64; e0 <= p.experts; e0 += 64)
        count += __builtin_amdgcn_readlane(scan_slots(p, pairs, e0, tile).sum, 63);
    return count;
}
// Tile number t of the experts' tiles: the expert (`experts + 1` past the last
// tile) and the tile's slots.
struct SlotTile {
    uint32_t expert, begin, end;
};
__device__ __forceinline__ SlotTile slot_tile(const Mx4Product &p, uint32_t pairs, uint32_t t, uint32_t tile, SlotScan s) {
    for (uint32_t e0 = 0;;) {
        const uint64_t over = __ballot(s.sum > t);
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            const uint32_t before = __builtin_amdgcn_readlane(s.sum - s.tiles, at);
            const uint32_t begin = __builtin_amdgcn_readlane(s.begin, at) + (t - before) * tile;
            const uint32_t end = __builtin_amdgcn_readlane(s.end, at);
            return {e0 + at, begin, min(begin + tile, end)};
        }
        t -= __builtin_amdgcn_readlane(s.sum, 63);
        e0 += 64;
        if (e0 > p.experts) return {p.experts + 1, 0, 0};
        s = scan_slots(p, pairs, e0, tile);
    }
}

// T x T tiles, four waves of T/2 x T/2 (256: eight of 128 x 64), slices of 256
// values: a slice's codes go global -> LDS directly, one slice ahead, with one
// barrier a slice, some of the next slice's transfers behind each of the steps'
// matrix instructions (all of them first, and the waves wait for their issue).
// The transfers are of whole lines (four times as many half lines arrive at 15
// TB/s, whole ones at 30), and a row's scales, 8 bytes a slice, come four slices
// at a time, or they would touch as many lines as the codes.
// 8192 x 8192 x 8192: 267 us, 4.11 PFLOP/s, the matrix cores busy in half of the
// cycles (as in a library's product of that size in BF16) at the 1.86 GHz that
// the card then runs at.  Left out of an earlier form of 291 us, the transfers
// gave 228, the products 242, and every line from L2 259: what bounds it is both
// together, and the power.
// A row's eight 16-byte blocks are stored in the order block ^ (row / 2 % 8):
// sixteen neighbouring rows' reads of one block cover all 64 banks.  The lanes'
// source addresses make the permutation.
// G > 1: G teams of four waves take a share of the tile's slices each, from
// stages of their own, and join their sums in LDS in the teams' order: tiles
// that leave CUs idle take 1 / G of the time (300 x 1000 x 4000 in tiles of 64:
// 10.8 us with one team, 7.7 with four; through a workspace and a launch
// of its own 10.9 to 15.7).
// With `splits` > 1 (dense products) workgroup z sums the slices [z, z + 1)
// slices / splits and writes part z of the output (FP32 parts in the
// workspace).
template <int T>
constexpr int kTeam = T == 256 ? 8 : 4;  // waves

template <int T, int G, Mode MODE, Mx4Type O>
__global__ __launch_bounds__(64 * G * kTeam<T>, T == 64 ? G : 2) void mx4_product_kernel(Mx4Product p, uint32_t tiles_m, uint32_t tiles_n,
                                                                         uint32_t splits) {
    constexpr int kWaves = kTeam<T>, kWavesN = kWaves / 2;
    constexpr int WM = T / 2, WN = T / kWavesN;     // a wave's part
    constexpr int BM = WM / 32, BN = WN / 32;       // in blocks of 32 x 32
    constexpr int kRowLoads = T / (8 * kWaves);     // 16-byte transfers of a lane per operand and slice
    struct Stage {
        uint8_t a[T * kCodeBytes], b[T * kCodeBytes];
    };
    constexpr int kGroup = 4 * kScaleBytes;  // a row's scales of four slices
    // an object each, so that reads of one are not held for transfers to another
    __shared__ __attribute__((aligned(1024))) Stage stage0[G], stage1[G];
    __shared__ __attribute__((aligned(1024))) uint8_t scale_words[G * 4 * T * kGroup];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % kWaves;
    const int team = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6) / kWaves;
    const Stage &s0 = stage0[team], &s1 = stage1[team];
    const uint8_t *scales_a = scale_words + team * 4 * T * kGroup, *scales_b = scales_a + 2 * T * kGroup;
    SlotScan scan;
    if constexpr (MODE == kRows) {
        // the tiles that there are, evenly over the XCDs
        scan = scan_slots(p, p.M, 0, T);
        tiles_m = slot_tiles(p, p.M, T, scan);
        if (blockIdx.x >= tiles_m * tiles_n) return;
    }
    int tm, tn, z;
    xcd_tile(static_cast<int>(tiles_m), static_cast<int>(tiles_n), static_cast<int>(splits), tm, tn, z);
    uint32_t m0 = tm * T, m_end = p.M, expert = 0, slice0 = 0, slices = p.slices;
    if constexpr (MODE == kDense) {
        slice0 = static_cast<uint32_t>(static_cast<uint64_t>(z) * p.slices / splits);
        slices = static_cast<uint32_t>(static_cast<uint64_t>(z + 1) * p.slices / splits) - slice0;
    } else if constexpr (MODE == kRows) {
        const SlotTile s = slot_tile(p, p.M, tm, T, scan);
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
    if (MODE != kDense && slices == 0) {  // uniform: nothing to sum, zeros
        const uint64_t first = MODE == kShared ? static_cast<uint64_t>(expert) * p.M : 0u;
        const float zero[8] = {};
        for (uint32_t c = tid; c < T * T / 8; c += blockDim.x) {
            const uint32_t m = m0 + c / (T / 8), n = tn * T + c % (T / 8) * 8;
            if (m >= m_end || n >= p.N) continue;
            uint64_t at = first + m;
            if constexpr (MODE == kRows) at = static_cast<uint32_t>(p.order[m]);
            store8<O>(p.out, at * p.ld + n, p.N - n, zero);
        }
        return;
    }
    // every team passes the same barriers, `turns` of them; one without a slice
    // transfers the last and multiplies none
    const uint32_t turns = (slices + G - 1) / G;
    uint32_t mine = slices;
    if constexpr (G > 1) {
        const uint32_t from = min(team * turns, slices), to = min(from + turns, slices);
        mine = to - from;
        slice0 += min(from, slices - 1);
        slices = max(mine, 1u);
    }
    const uint32_t n0 = tn * T;
    const uint64_t b_first = MODE == kRows ? static_cast<uint64_t>(min(expert, p.experts - 1)) * p.N : 0u;

    // This lane's rows and blocks of the transfers, as offsets from the tile's
    // first row (rows past the end repeat the last one; their results are not
    // stored).  Rows that the order chooses lie anywhere: 64 bits.
    const uint32_t pitch = p.slices * kCodeBytes, pitch_s = p.slices * kScaleBytes;
    const uint8_t *base_a = p.a.codes + static_cast<uint64_t>(slice0) * kCodeBytes;
    const uint8_t *base_sa = p.a.scales + static_cast<uint64_t>(slice0) * kScaleBytes;
    if constexpr (MODE != kRows) {
        base_a += static_cast<uint64_t>(m0) * pitch;
        base_sa += static_cast<uint64_t>(m0) * pitch_s;
    }
    const uint8_t *base_b = p.b.codes + (b_first + n0) * pitch + static_cast<uint64_t>(slice0) * kCodeBytes;
    const uint8_t *base_sb = p.b.scales + (b_first + n0) * pitch_s + static_cast<uint64_t>(slice0) * kScaleBytes;
    using Offset = std::conditional_t<MODE == kRows, uint64_t, uint32_t>;
    auto row_a = [&](uint32_t r) __attribute__((always_inline)) {
        const uint32_t row = min(m0 + r, m_end - 1);
        if constexpr (MODE == kRows) return static_cast<Offset>(static_cast<uint32_t>(p.order[row]) / p.per_token);
        else return static_cast<Offset>(row - m0);
    };
    auto row_b = [&](uint32_t r) __attribute__((always_inline)) { return min(n0 + r, p.N - 1) - n0; };
    const uint32_t block = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
    Offset oa[kRowLoads];
    uint32_t ob[kRowLoads];
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) {
        const uint32_t r = 8 * (kWaves * i + wave) + (lane >> 3);
        oa[i] = row_a(r) * pitch + 16 * block;
        ob[i] = row_b(r) * pitch + 16 * block;
    }
    // part 0 or 1 of the codes of slice k (past the end the last one's again,
    // which is not read: a branch here would part the matrix instructions from
    // their operands' reads)
    auto fetch_part = [&](const Stage &s, uint32_t k, int part) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        const uint64_t c = static_cast<uint64_t>(min(k, slices - 1)) * kCodeBytes;
        const uint8_t *pa = scalar<G>(base_a + c), *pb = scalar<G>(base_b + c);
#pragma unroll
        for (int i = 0; i < kRowLoads; ++i) {
            if (i / 3 != part) continue;
            dma16(pa + oa[i], s.a + 1024 * (kWaves * i + wave));
            dma16(pb + ob[i], s.b + 1024 * (kWaves * i + wave));
        }
        asm volatile("" ::: "memory");
    };
    // rows' part i of the scales of the four slices from k on, a lane four bytes
    // of the row whose codes it transfers (its offset in scales is a
    // sixteenth); words past the row's end repeat the last.  Rows eight apart
    // hold their words in another order, or they would share banks.
    auto fetch_scales = [&](uint32_t k, uint32_t i, Offset a, uint32_t b) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        const uint32_t word = 4 * min(2 * k + ((lane & 7) ^ (2 * (wave & 3))), 2 * slices - 1);
        const uint32_t to = (k & 4) / 4 * (T * kGroup) + 256 * (kWaves * i + wave);
        dma4(scalar<G>(base_sa) + ((a >> 4) - block + word), scales_a + to);
        dma4(scalar<G>(base_sb) + ((b >> 4) - block + word), scales_b + to);
        asm volatile("" ::: "memory");
    };
    // a part of the next four slices' with each slice
    auto next_scales = [&](uint32_t k) __attribute__((always_inline)) {
        const uint32_t i = k % kRowLoads;
        Offset a = oa[0];
        uint32_t b = ob[0];
#pragma unroll
        for (uint32_t j = 1; j < kRowLoads; ++j) {
            a = i == j ? oa[j] : a;
            b = i == j ? ob[j] : b;
        }
        fetch_scales((k & ~3u) + 4, i, a, b);
    };

    f32x16 acc[BM][BN] = {};
    const int wm = (wave / kWavesN) * WM, wn = (wave % kWavesN) * WN, row = lane & 31, half = lane >> 5;
    struct Frags {
        u32x4 a[BM], b[BN];
    };
    // A lane's block of step s lies at its first step's place xor 16 s, and its
    // scale word of slice k at that of slice 0 xor 8 (k % 4).  The places are
    // formed anew each time: kept, all steps' and stages' would not fit the
    // registers.
    const uint32_t place = row * kCodeBytes + 16 * ((4 * half) ^ ((row >> 1) & 7));
    const uint32_t place_s = row * kGroup + 4 * (half ^ (2 * ((row >> 3) & 3)));
    auto read = [&](Frags &f, const Stage &s, int step) __attribute__((always_inline)) {
        uint32_t at = place ^ (16 * step);
        asm volatile("" : "+v"(at));
        const uint8_t *pa = s.a + wm * kCodeBytes + at, *pb = s.b + wn * kCodeBytes + at;
#pragma unroll
        for (int i = 0; i < BM; ++i) f.a[i] = *reinterpret_cast<const u32x4 *>(pa + 32 * i * kCodeBytes);
#pragma unroll
        for (int j = 0; j < BN; ++j) f.b[j] = *reinterpret_cast<const u32x4 *>(pb + 32 * j * kCodeBytes);
    };
    uint32_t sa[2][BM], sb[2][BN];  // the scales of slice k in [k % 2]
    auto read_scales = [&](uint32_t k, int to) __attribute__((always_inline)) {
        uint32_t at = (k & 4) / 4 * (T * kGroup) + (place_s ^ (8 * (k & 3)));
        asm volatile("" : "+v"(at));
        const uint8_t *pa = scales_a + wm * kGroup + at, *pb = scales_b + wn * kGroup + at;
#pragma unroll
        for (int i = 0; i < BM; ++i) sa[to][i] = *reinterpret_cast<const uint32_t *>(pa + 32 * i * kGroup);
#pragma unroll
        for (int j = 0; j < BN; ++j) sb[to][j] = *reinterpret_cast<const uint32_t *>(pb + 32 * j * kGroup);
    };
    Frags f[2];
    // Slice k from `here`, whose first fragments and scales are in registers.
    // The barrier stands before the last step's products: once a wave has read
    // its fragments the stage is free for slice k + 2, and slice k + 1, whose
    // transfers have had a whole slice's time, is read while they run.
    auto slice = [&](const Stage &here, const Stage &other, uint32_t k, auto parity) __attribute__((always_inline)) {
        constexpr int P = decltype(parity)::value;
        if (G > 1 && k >= mine) {  // uniform in a wave
            stage_barrier<0>();
            return;
        }
        auto multiply = [&](auto st) __attribute__((always_inline)) {
            constexpr int S = decltype(st)::value;
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int j = 0; j < BN; ++j) acc[i][j] = mfma<S>(f[S & 1].a[i], f[S & 1].b[j], acc[i][j], sa[P][i], sb[P][j]);
        };
        read(f[1], here, 1);
        multiply(std::integral_constant<int, 0>{});
        fetch_part(other, k + 1, 1);
        next_scales(k);
        __builtin_amdgcn_sched_barrier(0);
        read(f[0], here, 2);
        multiply(std::integral_constant<int, 1>{});
        __builtin_amdgcn_sched_barrier(0);
        read(f[1], here, 3);
        multiply(std::integral_constant<int, 2>{});
        __builtin_amdgcn_sched_barrier(0);
        stage_barrier<0>();
        read(f[0], other, 0);
        read_scales(k + 1, P ^ 1);
        multiply(std::integral_constant<int, 3>{});
        __builtin_amdgcn_sched_barrier(0);
        // the sums stay on this side of the branch
#pragma unroll
        for (int i = 0; i < BM; ++i)
#pragma unroll
            for (int j = 0; j < BN; ++j) asm volatile("" : "+v"(acc[i][j]));
        if (k + 2 < slices) fetch_part(here, k + 2, 0);
    };
#pragma unroll
    for (uint32_t i = 0; i < kRowLoads; ++i) fetch_scales(0, i, oa[i], ob[i]);
    fetch_part(s0, 0, 0);
    fetch_part(s0, 0, 1);
    fetch_part(s1, 1, 0);
    stage_barrier<2 * (kRowLoads < 3 ? kRowLoads : 3)>();  // all but slice 1's
    read(f[0], s0, 0);
    read_scales(0, 0);
    uint32_t k = 0;
    for (; k + 2 <= turns; k += 2) {
        slice(s0, s1, k, std::integral_constant<int, 0>{});
        slice(s1, s0, k + 1, std::integral_constant<int, 1>{});
    }
    if (k < turns) slice(s0, s1, k, std::integral_constant<int, 0>{});
    const uint64_t out0 = MODE == kShared ? static_cast<uint64_t>(expert) * p.M : static_cast<uint64_t>(z) * p.M;
    // Out through LDS, 32 rows of the wave's at a time, so that a store covers
    // whole 16-byte pieces of a row.  The accumulators hold column lane % 32 of
    // a block and rows 8 (q / 4) + 4 (lane / 32) + q % 4; rows of the upper
    // half-wave have their columns' 32s swapped, or both would write one bank.
    constexpr int W = WN, swap = W >= 64 ? 32 : 0;
    constexpr int kPart = 32 * W;  // floats; half of a team's waves in either stage
    static_assert(kPart * 4 * kWaves <= 2 * sizeof(Stage), "the output's parts fit the stages");
    auto part_of = [&](int t, int w) __attribute__((always_inline)) {
        return reinterpret_cast<float *>((w < kWaves / 2 ? stage0[t].a : stage1[t].a)) + w % (kWaves / 2) * kPart;
    };
    stage_barrier<0>();
    float *stage = part_of(team, wave);
#pragma unroll
    for (int i = 0; i < BM; ++i) {
#pragma unroll
        for (int j = 0; j < BN; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q)
                stage[(8 * (q >> 2) + 4 * half + (q & 3)) * W + ((32 * j + row) ^ (swap * half))] = acc[i][j][q];
        // other lanes read what this one wrote: with one team only the wave's own
        if constexpr (G > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // The teams share a wave's rows out.  All of a lane's reads go out before
        // its first store, and no store waits for another (one piece after the
        // other took a third of the time of 16 products of 2752 x 2048 x 256).
        constexpr int kPieces = (kPart / 8 + 64 * G - 1) / (64 * G);
        auto piece = [&](int j) __attribute__((always_inline)) { return (lane + 64 * (team + G * j)) % (kPart / 8); };
        const bool some = 64 * team < kPart / 8;  // four teams have a piece for two
        float v[kPieces][8];
        uint64_t to[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int c = piece(j), r = c / (W / 8);
            const uint32_t m = min(m0 + wm + 32 * i + r, m_end - 1);
            if constexpr (MODE == kRows) to[j] = static_cast<uint32_t>(p.order[m]);
            else to[j] = out0 + m;
        }
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int c = piece(j), r = c / (W / 8), col = c % (W / 8) * 8;
            const int from = r * W + (col ^ (swap * ((r >> 2) & 1)));
            __builtin_memcpy(v[j], part_of(0, wave) + from, 32);
#pragma unroll
            for (int t = 1; t < G; ++t) {
                float u[8];
                __builtin_memcpy(u, part_of(t, wave) + from, 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] += u[e];
            }
        }
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int c = piece(j), r = c / (W / 8), col = c % (W / 8) * 8;
            const uint32_t m = m0 + wm + 32 * i + r, n = n0 + wn + col;
            if (some && m < m_end && n < p.N) store8<O>(p.out, to[j] * p.ld + n, p.N - n, v[j]);
        }
        // and all have read before the next rows take the place
        if constexpr (G == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else if (i + 1 < BM) __syncthreads();
    }
}

// The sum of the parts in order, rounded to the output's type; a lane takes
// eight columns.  A launch's time for the sizes that are split (37 x 4096, four
// parts of 606 KB, from L2: 2.5 us).
template <Mx4Type O>
__global__ __launch_bounds__(kThreads) void mx4_join_kernel(const float *__restrict__ parts, uint32_t splits, uint32_t M,
                                                            uint32_t N, void *__restrict__ out, uint64_t ld) {
    const uint32_t chunks = (N + 7) / 8;
    const uint64_t size = static_cast<uint64_t>(M) * N;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x, m = t / chunks;
    if (m >= M) return;
    const uint32_t n = 8 * static_cast<uint32_t>(t - m * chunks);
    float sum[8];
    load8<Mx4Type::F32>(parts, m * N + n, N - n, sum);
#pragma unroll 4
    for (uint32_t z = 1; z < splits; ++z) {
        float v[8];
        load8<Mx4Type::F32>(parts, z * size + m * N + n, N - n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
    store8<O>(out, m * ld + n, N - n, sum);
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A row's slice as v_mfma_scale_f32_16x16x128_f8f6f4 takes it: lane l has row
// l % 16 and, in step s of two, block 4 s + l / 16.
struct Slice16 {
    u32x4 codes[2];
    u32x2 scales;
    __device__ __forceinline__ void load(const Mx4Matrix &m, uint64_t row_slice, int g) {
        const uint8_t *p = m.codes + row_slice * kCodeBytes + 16 * g;
        codes[0] = *reinterpret_cast<const u32x4 *>(p);
        codes[1] = *reinterpret_cast<const u32x4 *>(p + 64);
        scales = *reinterpret_cast<const u32x2 *>(m.scales + row_slice * kScaleBytes);
    }
    __device__ __forceinline__ uint32_t scale(int s, int g) const { return scales[s] >> (8 * g); }
};

__device__ __forceinline__ f32x4_t mfma16(u32x4 a, u32x4 b, f32x4_t c, uint32_t sa, uint32_t sb) {
    const i32x8 a8 = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]), 0, 0, 0, 0};
    const i32x8 b8 = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, static_cast<int>(sa), 0, static_cast<int>(sb));
}

// Up to 16 rows of a: b is read once, straight into registers, by workgroups of
// 16 of its rows whose waves share the slices out in turn (a wave issues the
// loads of four slices before it uses the first), and the waves' sums are
// joined in LDS in the waves' order.
// X: the type of a dense x that every workgroup packs into LDS for itself while
// its first loads of b are in flight (kPacked: a is packed already).
// One row x 11008 x 4096: 8 us (24 MB, 4.7 us at the rate of a large copy), the
// launch and a wave's two rounds of loads; 64 pairs of 32 experts of 2752 x
// 4096: 33 to 36 us for the 160 MB of those that have any, HBM bound.
constexpr int kPacked = -1, kAhead = 4, kMostWaves = 16;  // the waves' sums: 16 KB

template <Mode MODE, Mx4Type O, int X>
__global__ __launch_bounds__(64 * kMostWaves) void mx4_few_rows_kernel(Mx4Product p, uint32_t tiles_n, uint32_t pairs,
                                                                       const void *x, uint64_t x_cols, uint64_t ldx) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const uint32_t tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
    uint32_t m0 = tm * 16, m_end = p.M, expert = 0, slices = p.slices;
    if constexpr (MODE == kRows) {
        const SlotTile s = slot_tile(p, pairs, tm, 16, scan_slots(p, pairs, 0, 16));
        if (s.expert > p.experts) return;  // uniform
        expert = s.expert;
        m0 = s.begin;
        m_end = s.end;
        if (expert == p.experts) slices = 0;  // slots of no expert: zero rows
    }
    const uint32_t n0 = tn * 16;
    const uint64_t b_first = MODE == kRows ? static_cast<uint64_t>(min(expert, p.experts - 1)) * p.N : 0u;
    uint64_t a_row = min(m0 + r, m_end - 1);  // its first slice, as b's
    if constexpr (MODE == kRows) a_row = static_cast<uint32_t>(p.order[a_row]) / p.per_token;
    a_row *= p.slices;
    const uint64_t b_row = (b_first + min(n0 + r, p.N - 1)) * p.slices;

    Slice16 a[kAhead], b[kAhead];
    auto load = [&](uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t k = min(k0 + u * waves, slices - 1);  // past the end: the last slice again, not used
            b[u].load(p.b, b_row + k, g);
            if constexpr (X == kPacked) a[u].load(p.a, a_row + k, g);
        }
    };
    uint32_t k0 = wave;
    if (k0 < slices) load(k0);
    if constexpr (X != kPacked) {
        constexpr Mx4Type T = static_cast<Mx4Type>(X == kPacked ? 0 : X);
        constexpr int size = T == Mx4Type::F32 ? 4 : 2;
        const uint32_t blocks = p.slices * 8, all = p.M * blocks;
        for (uint32_t t = tid; t < all; t += blockDim.x) {
            const uint32_t row = t / blocks, blk = t - row * blocks;
            const uint8_t *from = static_cast<const uint8_t *>(x) + static_cast<uint64_t>(row) * ldx * size;
            Eight<T> v[4];
            if (32ull * blk + 32 <= x_cols) {
                __builtin_memcpy(v, from + 32ull * blk * size, sizeof v);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q].load(from, 32ull * blk + 8 * q, x_cols);
            }
            const uint32_t byte = mx4_scale_byte(f32_bits<T>(max(max(v[0].top(), v[1].top()), max(v[2].top(), v[3].top()))));
            u32x4 c = {0, 0, 0, 0};
            if (byte != 255u) {
#pragma unroll
                for (int q = 0; q < 4; ++q) c[q] = v[q].codes(mx4_power(byte));
            }
            *reinterpret_cast<u32x4 *>(lds + 16 * t) = c;
            lds[16 * all + t] = static_cast<uint8_t>(byte);
        }
        __syncthreads();
    }
    f32x4_t acc = {};
    while (k0 < slices) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t k = k0 + u * waves;
            if (k >= slices) break;  // uniform
            if constexpr (X != kPacked) {
                const Mx4Matrix packed{lds, lds + 16 * 8 * p.M * p.slices};
                a[u].load(packed, a_row + k, g);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) acc = mfma16(a[u].codes[s], b[u].codes[s], acc, a[u].scale(s, g), b[u].scale(s, g));
        }
        k0 += kAhead * waves;
        if (k0 < slices) load(k0);
    }
    if constexpr (X != kPacked) __syncthreads();  // the packed x is done with
    // lane: column n = lane % 16, rows 4 (lane / 16) + q
    float *part = reinterpret_cast<float *>(lds);  // [wave][16][16]
#pragma unroll
    for (int q = 0; q < 4; ++q) part[(wave * 16 + 4 * g + q) * 16 + r] = acc[q];
    __syncthreads();
    for (uint32_t t = tid; t < 256; t += blockDim.x) {
        const uint32_t m = m0 + t / 16, n = n0 + t % 16;
        if (m >= m_end || n >= p.N) continue;
        float sum = part[t];
        for (int w = 1; w < waves; ++w) sum += part[w * 256 + t];
        uint64_t at = m;
        if constexpr (MODE == kRows) at = static_cast<uint32_t>(p.order[m]);
        store_value<O>(p.out, at * p.ld + n, sum);
    }
}

// x is packed again in every workgroup rather than once in a launch of its own
// (some 3 us) as long as it fits their LDS and what they read of it together
// (`kPackReads` values) comes from L2 in less than that.
constexpr uint32_t kPackRows = 16, kPackBytes = 32768;
constexpr uint64_t kPackReads = 4ull << 20;
// Rows up to which b is streamed (16 x 4096 x 11008: 10.1 us; in tiles of 64 37
// rows take 13.3).
constexpr uint32_t kFewRows = 16;

constexpr const char *kTooLarge = "mx4 product: too large";
unsigned few_rows_waves(const Mx4Product &p) {
    return std::min<unsigned>(kMostWaves, std::max(1u, (p.slices + kAhead - 1) / kAhead));
}

template <Mode MODE, int X>
void few_rows(const Mx4Product &p, uint64_t tiles_m, uint32_t pairs, const void *x, uint64_t x_cols, uint64_t ldx,
              hipStream_t stream) {
    const uint64_t tiles_n = ceil_div(p.N, 16);
    const unsigned waves = few_rows_waves(p), grid = grid_of(tiles_n * tiles_m, 64 * waves, kTooLarge);
    const unsigned lds = std::max(waves * 1024, X == kPacked ? 0u : p.M * p.slices * 136);
    by_type(p.type, [&](auto t) {
        mx4_few_rows_kernel<MODE, decltype(t)::value, X>
            <<<grid, 64 * waves, lds, stream>>>(p, static_cast<uint32_t>(tiles_n), pairs, x, x_cols, ldx);
    });
}

}  // namespace

bool mx4_packs_on_the_way(uint64_t m, uint64_t n, uint64_t slices) {
    return m <= kPackRows && m * slices * 136 <= kPackBytes && m * slices * kMx4Slice * ceil_div(n, 16) <= kPackReads;
}

void launch_mx4_product_of(const void *x, Mx4Type x_type, uint64_t x_cols, uint64_t ldx, const Mx4Product &p,
                           hipStream_t stream) {
    if (p.M == 0 || p.N == 0) return;
    by_type(x_type, [&](auto t) {
        few_rows<kDense, static_cast<int>(decltype(t)::value)>(p, 1, 0, x, x_cols, ldx, stream);
    });
    BSQ_HIP(hipGetLastError());
}

namespace {

// How a product is cut.  Measured in us (M x N x K, tile . teams):
//   8192 x 4096 x 4096    128.1 91.4  128.2 113    256 75.4
//   2048 x 4096 x 4096    64.1 36.8   128.1 24.6   128.2 28.9   256 31.4
//   1024 x 4096 x 4096    64.1 21.1   64.2 21.3    128.1 16.7   128.2 15.8
//    512 x 4096 x 4096    64.1 13.5   64.2 12.3    64.4 15.7    128.2 14.1
//    256 x 4096 x 4096    64.1 11.8   64.2 9.0     64.4 8.7     128.2 13.6
//   2000 x  300 x  512    64.1 4.0    64.2 4.0     64.4 4.9     128.2 6.3
// Teams as long as every workgroup still finds a CU of its own; tiles of 256
// where their rounds over the CUs cost less (a round of one a CU 2.4 us a
// slice, of two 128s a CU 1.44).
bool large_tiles(uint64_t rows128, uint64_t rows256, uint64_t N) {
    const uint64_t cus = static_cast<uint64_t>(cu_count());
    return 2.4 * ceil_div(ceil_div(rows256, 256) * ceil_div(N, 256), cus) <
           1.44 * ceil_div(ceil_div(rows128, 128) * ceil_div(N, 128), 2 * cus);
}
struct Plan {
    uint32_t tile, tiles_m, tiles_n, teams, splits;
    uint64_t bytes;
};
Plan plan_of(uint32_t M, uint32_t N, uint32_t slices) {
    const uint64_t cus = static_cast<uint64_t>(cu_count());
    auto tiles = [&](uint64_t t) { return ceil_div(M, t) * ceil_div(N, t); };
    Plan q{128, 0, 0, 1, 1, 0};
    if (tiles(128) > 2 * cus) {
        if (large_tiles(M, M, N)) q.tile = 256;
    } else if (tiles(64) > 2 * cus) {
        q.teams = tiles(128) <= cus && slices > 1 ? 2 : 1;
    } else {
        q.tile = 64;
        q.teams = slices == 1 ? 1 : tiles(64) > cus || slices < 8 ? 2 : 4;
    }
    if (q.tile == 64 && q.teams == 4) {
        // more workgroups for a long shared axis: a turn of four slices 1.6 us,
        // against the join's launch and the parts' way to memory and back (37
        // x 4096 x 11008: 21.2 us with one split, 13.3 with 4; 128 x 128 x
        // 60000: 70 and, with 8, 15.8)
        double best = 0.0;
        for (uint32_t s = 1; s <= 16 && tiles(64) * s <= 2 * cus; s *= 2) {
            const double t = 1.6 * ceil_div(slices, 4 * s) + (s > 1 ? 4.0 + s * (8.0 * M * N / 2.5e6) : 0.0);
            if (s == 1 || t < best) {
                best = t;
                q.splits = s;
            }
        }
    }
    q.tiles_m = static_cast<uint32_t>(ceil_div(M, q.tile));
    q.tiles_n = static_cast<uint32_t>(ceil_div(N, q.tile));
    q.bytes = q.splits > 1 ? static_cast<uint64_t>(q.splits) * M * N * 4 : 0;
    return q;
}

// A product's kernel and its grid; a tile of 16 stands for few rows.
struct Cut {
    uint32_t tile, teams, splits;
    uint64_t tiles_m, tiles_n, bytes;
};
Cut cut_of(const Mx4Product &p) {
    auto cut = [&](uint32_t tile, uint32_t teams, uint64_t tiles_m) {
        return Cut{tile, teams, 1, tiles_m, ceil_div(p.N, tile), 0};
    };
    if (p.shared_slots) {
        // (480 tokens to 4 experts, 176 x 338: 256 14.2 us, 64 4.9; 4096 pairs of
        // 16 experts, 2752 x 2048: 256 66, 128 70, where the 180 MB written take
        // some 35)
        const uint64_t cus = static_cast<uint64_t>(cu_count());
        auto of = [&](uint64_t t) { return p.experts * ceil_div(p.M, t) * ceil_div(p.N, t); };
        const uint32_t tile = of(128) <= cus ? 64 : of(256) <= 2 * cus ? 128 : 256;
        return cut(tile, 1, ceil_div(p.M, tile));
    }
    if (p.offsets != nullptr) {
        // M: the pairs; every expert's tiles, and those of the pairs of none, none
        // of them empty.  What the cut goes by: half a tile an expert left over.
        auto of = [&](uint64_t t) { return std::min<uint64_t>(p.M, ceil_div(p.M, t) + p.experts + 1); };
        // (us of the layer, 2752 x 4096, with 16 and with 64: 16 pairs of 32 experts
        // 26 and 26, of one 13 and 18; 128 of 32 56 and 54, of one 26 and 19; 512 of
        // 32 90 and 60, of one 71 and 23)
        if (p.M / p.experts <= 16) return cut(16, 1, of(16));
        const uint64_t cus = static_cast<uint64_t>(cu_count());
        auto rows = [&](uint64_t t) { return p.M + t / 2 * p.experts; };
        auto count = [&](uint64_t t) { return ceil_div(rows(t), t) * ceil_div(p.N, t); };
        if (count(64) <= 2 * cus && p.slices > 1) return cut(64, 2, of(64));
        if (count(128) <= cus || p.M / p.experts <= 64) return cut(64, 1, of(64));
        // (us: 16384 pairs of 32 experts, 2752 x 4096 to BF16 with 256 156 to 168,
        // with 128 177 to 193; 4096 of 16 to FP32, 2752 x 2048 with 128 45, with
        // 256 57, 2048 x 2752 47 and 42)
        const uint32_t tile = large_tiles(rows(128), rows(256), p.N) ? 256 : 128;
        return cut(tile, 1, of(tile));
    }
    if (p.M <= kFewRows) return cut(16, 1, 1);
    const Plan q = plan_of(p.M, p.N, p.slices);
    return {q.tile, q.teams, q.splits, q.tiles_m, q.tiles_n, q.bytes};
}
uint32_t threads_of(const Cut &c, const Mx4Product &p) {
    return 64 * (c.tile == 16 ? few_rows_waves(p) : c.teams * (c.tile == 256 ? kTeam<256> : kTeam<64>));
}

template <int T, int G, Mode MODE>
void tiles(const Mx4Product &p, const Cut &c, hipStream_t stream) {
    const unsigned groups = grid_of(c.tiles_m * c.tiles_n * c.splits, 64 * G * kTeam<T>, kTooLarge);
    const dim3 g(groups, MODE == kShared ? p.experts : 1);
    by_type(p.type, [&](auto t) {
        mx4_product_kernel<T, G, MODE, decltype(t)::value><<<g, 64 * G * kTeam<T>, 0, stream>>>(
            p, static_cast<uint32_t>(c.tiles_m), static_cast<uint32_t>(c.tiles_n), c.splits);
    });
}

}  // namespace

uint64_t mx4_product_workspace(uint32_t M, uint32_t N, uint32_t slices) {
    return M <= kFewRows || N == 0 ? 0 : plan_of(M, N, slices).bytes;
}

void check_mx4_product(const Mx4Product &p) {
    if (p.M == 0 || p.N == 0) return;
    const Cut c = cut_of(p);
    grid_of(c.tiles_m * c.tiles_n * c.splits, threads_of(c, p), kTooLarge);
}

void launch_mx4_product(const Mx4Product &p, void *workspace, uint64_t workspace_bytes, hipStream_t stream) {
    if (p.M == 0 || p.N == 0) return;
    const Cut c = cut_of(p);
    if (p.shared_slots) {
        if (c.tile == 64) tiles<64, 1, kShared>(p, c, stream);
        else if (c.tile == 128) tiles<128, 1, kShared>(p, c, stream);
        else tiles<256, 1, kShared>(p, c, stream);
    } else if (p.offsets != nullptr) {
        if (c.tile == 16) few_rows<kRows, kPacked>(p, c.tiles_m, p.M, nullptr, 0, 0, stream);
        else if (c.tile == 64 && c.teams == 2) tiles<64, 2, kRows>(p, c, stream);
        else if (c.tile == 64) tiles<64, 1, kRows>(p, c, stream);
        else if (c.tile == 128) tiles<128, 1, kRows>(p, c, stream);
        else tiles<256, 1, kRows>(p, c, stream);
    } else if (c.tile == 16) {
        few_rows<kDense, kPacked>(p, 1, 0, nullptr, 0, 0, stream);
    } else {
        BSQ_REQUIRE(workspace_bytes >= c.bytes, "mx4 product: workspace too small");
        Mx4Product part = p;
        if (c.splits > 1) {
            part.out = workspace;
            part.type = Mx4Type::F32;
            part.ld = p.N;
        }
        if (c.tile == 256) tiles<256, 1, kDense>(part, c, stream);
        else if (c.tile == 128 && c.teams == 2) tiles<128, 2, kDense>(part, c, stream);
        else if (c.tile == 128) tiles<128, 1, kDense>(part, c, stream);
        else if (c.teams == 4) tiles<64, 4, kDense>(part, c, stream);
        else if (c.teams == 2) tiles<64, 2, kDense>(part, c, stream);
        else tiles<64, 1, kDense>(part, c, stream);
        if (c.splits > 1) {
            by_type(p.type, [&](auto t) {
                const uint64_t grid = ceil_div(p.M * ceil_div(p.N, 8), kThreads);
                mx4_join_kernel<decltype(t)::value><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(
                    static_cast<const float *>(workspace), c.splits, p.M, p.N, p.out, p.ld);
            });
        }
    }
    BSQ_HIP(hipGetLastError());
}

}  // namespace bsq
