// Attention over the paged MX4 cache: single tokens and a few queries a request
// (kv4_attention.hpp).  A source for each number of pieces instantiates it, as the
// compiler takes its time over the kernels.
//
// Long contexts are bound by HBM: 8 requests of 40 to 90 thousand keys, 32 query
// heads on 8 of 128, take 107 us with the join, 5.0 TB/s of the 5.07 that a large
// copy reaches.  Of ragged ones (128 requests of 16 to 16384 keys, 76 us, 4.4 TB/s)
// and short ones (16 of 400 to 1200, 15.0 us) what a tile costs beside its keys is
// the rest; each further step of 32 keys adds a wave alone on its SIMD some 0.8 us
// (least shares of 4 to 12 steps, 15.8 to 22.3 us); keys are asked for one step ahead.
// A form with a workgroup's waves on one tile, joined in LDS, took 89 us for the ragged
// and 15.5 for the short ones; 9 requests of 5 queries over 100 to 5000 keys, 12 heads
// of 64 in FP32, took 15.4 with it and take 18.4 with waves as shares.
#pragma once

#include "kv4_attention.hpp"

namespace bsq {
namespace {

__device__ __forceinline__ uint32_t first_key(const AttentionArgs &a, const Request &q) {
    return a.window == 0 ? 0u : static_cast<uint32_t>(max(q.past() + 1 - static_cast<int64_t>(a.window), static_cast<int64_t>(0))) & ~(kStep - 1);
}
__device__ __forceinline__ uint32_t spans_of(const AttentionArgs &a, const Request &q) {
    const uint32_t first = first_key(a, q), length = static_cast<uint32_t>(q.length);
    return length > first ? (length - first + ((1u << a.span) - 1)) >> a.span : 1u;
}
__device__ __forceinline__ uint32_t tiles_of(const AttentionArgs &a, const Request &q) {
    const uint64_t rows = static_cast<uint64_t>(q.count) * a.group;
    return rows > a.few ? 0u : static_cast<uint32_t>((rows + kTileRows - 1) / kTileRows);
}

template <int NB>
struct Shape {
    static constexpr int kLane = NB == 1 ? 2 : NB == 2 ? 4 : NB <= 4 ? 8 : 16;  // values of a lane's channels
    static constexpr int kLanes = 32 * NB / kLane;                              // of 16 that hold channels
    static constexpr int kWords = kLane <= 8 ? 1 : 2;
    // words of a lane's key scales: a lane has 8 NB channels from 8 NB g on
    static constexpr int kScales = NB % 4 == 0 ? NB / 4 : NB <= 2 ? 1 : NB;
};

// 32 keys and values as a lane takes them.  Lane l = 16 g + i.  Keys: the row of
// token 16 a + 4 (i % 4) + i / 4 of the two sixteens a, channels [8 NB g, 8 NB (g
// + 1)).  The products' lane then holds, for query i, the tokens 16 a + 4 r + g =
// 4 j + g with j = 4 a + r: the eight that it holds of the values' rows, channels
// [kLane i, kLane (i + 1)), so the weights stay where they are.
template <int NB>
struct Tile {
    using S = Shape<NB>;
    static constexpr uint32_t kRow = 16 * NB;  // bytes of a token's codes
    uint32_t k[2][NB], ks[2][S::kScales], v[8][S::kWords], vs[2];
    uint32_t bad;  // bit a: the sixteen is on no page

    // a lane's places from those of a sixteen's first token
    struct Places {
        uint32_t k, ks[S::kScales], v, vs;
        __device__ __forceinline__ explicit Places(uint32_t lane) {
            const uint32_t g = lane >> 4, i = lane & 15, c = min(i, static_cast<uint32_t>(S::kLanes - 1));
            k = (4 * (i & 3) + (i >> 2)) * kRow + g * (4 * NB);
#pragma unroll
            for (int u = 0; u < S::kScales; ++u) {
                const uint32_t b = NB % 4 == 0 ? g * (NB / 4) + u : (g * NB + u) >> 2;
                ks[u] = (i >> 2) * (4 * NB) + 4 * b + (i & 3);
            }
            v = g * kRow + c * (S::kLane / 2);
            vs = g * (4 * NB) + 4 * ((c * S::kLane) >> 5);
        }
    };

    // head: of head h on page 0; the addresses up to a lane's places are scalar
    __device__ __forceinline__ void load(const Kv4Cache &cache, const uint8_t *head, uint32_t page_bytes, uint32_t t, uint32_t id0,
                                         uint32_t id1, const Places &at) {
        const uint32_t bad0 = id0 >= cache.count ? 1u : 0u, bad1 = id1 >= cache.count ? 2u : 0u;
        bad = bad0 | bad1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t id = (s ? bad1 : bad0) ? 0u : (s ? id1 : id0);
            const uint32_t in = (t + 16 * s) & (cache.page() - 1);
            const uint8_t *p = head + static_cast<uint64_t>(id) * page_bytes;
            const uint8_t *kp = p + in * kRow, *vp = kp + (kRow << cache.shift);
            const uint8_t *ksp = p + (2 * kRow << cache.shift) + in * NB, *vsp = ksp + (NB << cache.shift);
            __builtin_memcpy(k[s], __builtin_assume_aligned(kp + at.k, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), 4 * NB);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint8_t *q = vp + at.v + 4 * r * kRow;
                if constexpr (S::kLane == 2) v[4 * s + r][0] = *q;
                else if constexpr (S::kLane == 4) v[4 * s + r][0] = *reinterpret_cast<const uint16_t *>(q);
                else __builtin_memcpy(v[4 * s + r], __builtin_assume_aligned(q, 4 * S::kWords), 4 * S::kWords);
            }
#pragma unroll
            for (int u = 0; u < S::kScales; ++u) ks[s][u] = ksp[at.ks[u]];
            vs[s] = *reinterpret_cast<const uint32_t *>(vsp + at.vs);
        }
    }
};

// A wave's state for its tile of 16 queries: lane (g, i) has query i's reference,
// its share of the sum, and of the channels' sums those of kLane (4 g + r) + c.
template <int NB, int P>
struct Rows {
    using S = Shape<NB>;
    u32x4 q[P][NB];
    f32x4 o[S::kLane];
    float top, base, sum;  // base: top, 0 where that is minus infinity

    // A lane's words of queries, asked for ahead of begin(): those of 16 bits.
    struct Ahead {
        uint32_t w[NB][4];
    };
    __device__ __forceinline__ static uint64_t query_at(const AttentionArgs &a, const Request &rq, uint32_t h, uint32_t row) {
        const uint64_t token = static_cast<uint32_t>(rq.first) + row / a.group;
        return token * a.ldq + static_cast<uint64_t>(h * a.group + row % a.group) * a.cache.dim;
    }
    __device__ __forceinline__ static void ask(const AttentionArgs &a, Ahead &ahead, const Request &rq, uint32_t h, uint32_t row0,
                                               uint32_t rows, uint32_t lane) {
        if constexpr (P < 3) {
            const uint32_t g = lane >> 4, i = lane & 15, dim = a.cache.dim;
            const uint16_t *from = reinterpret_cast<const uint16_t *>(a.q) + query_at(a, rq, h, row0 + i);
#pragma unroll
            for (int s = 0; s < NB; ++s) {
                const uint32_t c = (g * NB + s) * 8;
                u32x4 w = {0, 0, 0, 0};
                if (i < rows && c + 8 <= dim) {
                    __builtin_memcpy(&w, from + c, 16);
                } else if (i < rows && c < dim) {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e)
                        if (c + e < dim) w[e >> 1] |= static_cast<uint32_t>(from[c + e]) << (16 * (e & 1));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) ahead.w[s][e] = w[e];
            }
        }
    }
    __device__ __forceinline__ void begin(const AttentionArgs &a, const Ahead &ahead, const Request &rq, uint32_t h, uint32_t row0,
                                          uint32_t rows, uint32_t lane) {
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if constexpr (P == 1) {  // BF16 as it is, but infinities NaN as in pieces(): 0x7F80 | 1
                constexpr mx4_u16x2 kFinite = {0x7F7F, 0x7F7F};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = ahead.w[s][e];
                    const mx4_u16x2 above = __builtin_elementwise_sub_sat(__builtin_bit_cast(mx4_u16x2, w & 0x7FFF7FFFu), kFinite);
                    q[0][s][e] = (a.negate ? w ^ 0x80008000u : w) | __builtin_bit_cast(uint32_t, above);
                }
                continue;
            }
            if constexpr (P == 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t w = ahead.w[s][e >> 1] >> (16 * (e & 1)) & 0xFFFFu;
                    x[e] = a.q_type == Mx4Type::BF16 ? bf16_value(w) : f16_value(w);
                }
            } else {
                const uint32_t g = lane >> 4, i = lane & 15, c = (g * NB + s) * 8;
                if (i < rows && c < a.cache.dim)
                    by_device_type(a.q_type, [&](auto t) {
                        load8<decltype(t)::value>(a.q, query_at(a, rq, h, row0 + i) + c, a.cache.dim - c, x);
                    });
            }
            if (a.negate) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = -x[e];
            }
            u32x4 w[P];
            pieces<P, true>(x, w);
#pragma unroll
            for (int p = 0; p < P; ++p) q[p][s] = w[p];
        }
#pragma unroll
        for (int c = 0; c < S::kLane; ++c) o[c] = f32x4{0, 0, 0, 0};
        top = -__builtin_inff();
        base = sum = 0.0f;
    }

    // lim, low: the query sees the tokens [low, lim).  any_lim, any_low: some of
    // the tile's queries see those.  masked: not all of them see all.
    __device__ __forceinline__ void step(const AttentionArgs &a, const Tile<NB> &tile, uint32_t t, uint32_t lane, bool masked,
                                         int32_t lim, int32_t low, int32_t any_lim, int32_t any_low, bool mixed) {
        const uint32_t g = lane >> 4;
        f32x4 x[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const float scale = __uint_as_float(tile.ks[s][NB % 4 == 0 ? u / 4 : NB <= 2 ? 0 : u] << 23);
                const uint32_t w = tile.k[s][u];
                const u32x4 k = {cvt(w, scale, 0), cvt(w, scale, 1), cvt(w, scale, 2), cvt(w, scale, 3)};
#pragma unroll
                for (int p = 0; p < P; ++p) x[s] = mfma(k, q[p][u], x[s]);
            }
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = x[j >> 2][j & 3] * a.factor;
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int32_t at = static_cast<int32_t>(t + 4 * j + g);
                if (at >= lim || at < low || (tile.bad >> (j >> 2) & 1)) w[j] = -__builtin_inff();
            }
        }
        float high = w[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) high = fmaxf(high, w[j]);
        if (__any(high > top + kSlack)) {
            high = fmaxf(high, __shfl_xor(high, 16));
            high = fmaxf(high, __shfl_xor(high, 32));
            const float now = fmaxf(top, high), keep = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            sum *= keep;
#pragma unroll
            for (int c = 0; c < S::kLane; ++c) o[c] *= keep;
            top = now;
            base = now == -__builtin_inff() ? 0.0f : now;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = __builtin_amdgcn_exp2f(w[j] - base);
            sum += w[j];
        }
        u32x4 pw[P];
        pieces<P>(w, pw);

        uint32_t v[8][S::kWords], vs[2] = {tile.vs[0], tile.vs[1]};
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int d = 0; d < S::kWords; ++d) v[j][d] = tile.v[j][d];
        if (masked) {
            // what no query sees may hold anything, NaN among it
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int32_t at = static_cast<int32_t>(t + 4 * j + g);
                uint32_t byte = (vs[j >> 2] >> (8 * (j & 3))) & 0xFFu;
                if (at >= any_lim || at < any_low || (tile.bad >> (j >> 2) & 1)) {
                    byte = 127;
#pragma unroll
                    for (int d = 0; d < S::kWords; ++d) v[j][d] = 0;
                }
                if (mixed) poison(a, byte, v[j], t + 4 * j, lane, lim, low);
                vs[j >> 2] = (vs[j >> 2] & ~(0xFFu << (8 * (j & 3)))) | byte << (8 * (j & 3));
            }
        }
        float scale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) scale[j] = __uint_as_float(((vs[j >> 2] >> (8 * (j & 3))) & 0xFFu) << 23);
#pragma unroll
        for (int c = 0; c < S::kLane; c += 2) {
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t x0 = cvt(v[j][c >> 3], scale[j], (c >> 1) & 3), x1 = cvt(v[j + 1][c >> 3], scale[j + 1], (c >> 1) & 3);
                even[j >> 1] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
                odd[j >> 1] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                o[c] = mfma(even, pw[p], o[c]);
                o[c + 1] = mfma(odd, pw[p], o[c + 1]);
            }
        }
    }

    // A NaN block of values that some of the tile's queries see and others do not:
    // the products would give 0 times NaN to those that do not.  It leaves the
    // products and goes into the sums of those that do.
    __device__ __forceinline__ void poison(const AttentionArgs &a, uint32_t &byte, uint32_t v[S::kWords], uint32_t t0, uint32_t lane,
                                           int32_t lim, int32_t low) {
        uint64_t nan = __ballot(byte == 255u);
        if (nan == 0) return;
        if (byte == 255u) {
            byte = 127;
#pragma unroll
            for (int d = 0; d < S::kWords; ++d) v[d] = 0;
        }
        while (nan != 0) {
            const uint32_t from = static_cast<uint32_t>(__builtin_ctzll(nan));
            nan &= nan - 1;
            const int32_t at = static_cast<int32_t>(t0 + (from >> 4));
            const uint32_t block = ((from & 15) * S::kLane) >> 5;
            if (at >= lim || at < low) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (((4 * (lane >> 4) + r) * S::kLane) >> 5 == block) {
#pragma unroll
                    for (int c = 0; c < S::kLane; ++c) o[c][r] = __builtin_nanf("");
                }
        }
    }
};

// Each wave takes an equal share of all units of all requests' tiles: every tile of
// every head, in order, so that contexts of any lengths keep all CUs busy alike.
// A tile whose keys lie in one share is written at once; of one whose do not, each
// share leaves its sums, and the join below adds them.  Waves need nothing of one
// another: no LDS, no barriers.
template <int NB, int P>
__global__ __launch_bounds__(kFewThreads, NB <= 4 ? 2 : 1) void kv4_attention_kernel(AttentionArgs a, uint32_t waves) {
    using S = Shape<NB>;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t share = blockIdx.x * kFewWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t heads = a.cache.heads;
    if (share >= waves) return;

    // a lane's run of requests, and the units before it
    const uint32_t per = (a.requests + 63) / 64;
    const uint32_t r_begin = min(lane * per, a.requests), r_end = min(r_begin + per, a.requests);
    Request own{0, 0, 0};  // with one request a lane
    uint64_t units_here = 0;
    for (uint32_t i = r_begin; i < r_end; ++i) {
        own = load_request(a, i);
        units_here += static_cast<uint64_t>(tiles_of(a, own)) * (spans_of(a, own) + kExtra);
    }
    units_here *= heads;
    // The host has seen to it that all fit 31 bits, unless starts overlap: those that
    // then do not are no work.
    const bool too_many = __any(units_here >= 1u << 25) && [&] {
        uint64_t sum = units_here;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        return sum >= 1ull << 31;
    }();
    const uint32_t mine = too_many ? 0u : static_cast<uint32_t>(units_here);
    const uint32_t up_to = wave_prefix(mine), total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(up_to), 63));
    // no share is empty but those behind the last: a split tile's lie side by side
    const uint32_t shares = min(max(total / kLeast, min(total, 1u)), waves);
    if (share >= shares) {
        if (lane == 0) a.splits[share].parts = 0;
        return;
    }
    // the first `more` shares have `even` + 1 units, the others `even`
    const uint32_t even = total / shares, more = total - even * shares;
    const uint32_t begin = share * even + min(share, more), end = begin + even + (share < more ? 1 : 0);
    const auto share_of = [&](uint32_t x) {
        const uint32_t longer = more * (even + 1);
        return x < longer ? x / (even + 1) : more + (x - longer) / even;
    };
    const auto request = [&](uint32_t i) {
        if (per > 1) return load_request(a, i);
        const int at = static_cast<int>(i);
        return Request{__builtin_amdgcn_readlane(own.length, at), __builtin_amdgcn_readlane(own.first, at),
                       __builtin_amdgcn_readlane(own.count, at)};
    };
    const uint64_t behind = __ballot(begin < up_to);
    const uint32_t in_lane = behind ? static_cast<uint32_t>(__builtin_ctzll(behind)) : 0u;

    // where this share is: the unit `x`, unit `u` of tile `tile` of head `h`
    uint32_t r = in_lane * per, x = begin, h = 0, tile = 0, u = 0;
    Request rq = request(r);
    uint32_t units = spans_of(a, rq) + kExtra, tiles = tiles_of(a, rq);
    {
        uint32_t base = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(up_to - mine), static_cast<int>(in_lane)));
        while (x - base >= tiles * units * heads && r + 1 < a.requests) {
            base += tiles * units * heads;
            rq = request(++r);
            units = spans_of(a, rq) + kExtra, tiles = tiles_of(a, rq);
        }
        if (tiles > 0) {
            const uint32_t at = (x - base) / units;
            u = (x - base) - at * units;
            h = at / tiles;
            tile = at - h * tiles;
        }
    }

    // a tile, or a part of one, that this share holds
    struct Work {
        Request rq;
        uint32_t r, h, row0, count;
        uint32_t last;      // the tile's last unit
        bool first, whole;  // it holds the first keys, all of them
        int32_t from, to;   // keys
    };
    const int32_t window = static_cast<int32_t>(min(a.window, 0x7FFFFFFFu));
    const auto query_of = [&](const Request &q, uint32_t row) { return q.count == 1 ? 0 : static_cast<int32_t>(row / a.group); };
    const auto lim_of = [&](const Request &q, int32_t query) { return a.causal ? q.past() + query + 1 : q.length; };
    const auto low_of = [&](const Request &q, int32_t query) { return window ? max(q.past() + query + 1, 0) - window : 0; };
    const auto next = [&](Work &w) __attribute__((always_inline)) {
        while (x < end) {
            if (h >= heads || tiles == 0) {
                if (++r >= a.requests) return false;  // starts that overlap
                rq = request(r);
                units = spans_of(a, rq) + kExtra, tiles = tiles_of(a, rq);
                h = tile = u = 0;
                continue;
            }
            const uint32_t u0 = u, u1 = min(units, u0 + (end - x));
            w.h = h, w.row0 = tile * kTileRows, w.last = x + (units - u0) - 1;
            x += u1 - u0;
            u = u1;
            if (u1 == units) {
                u = 0;
                if (++tile == tiles) tile = 0, ++h;
            }
            // the units ahead of the keys come first
            const uint32_t j0 = max(u0, kExtra) - kExtra, j1 = max(u1, kExtra) - kExtra;
            if (j1 <= j0) continue;
            w.rq = rq, w.r = r;
            w.count = min(kTileRows, static_cast<uint32_t>(rq.count) * a.group - w.row0);
            w.first = j0 == 0, w.whole = j0 == 0 && u1 == units;
            const uint32_t t0 = first_key(a, rq);
            const int32_t any_lim = lim_of(rq, query_of(rq, w.row0 + w.count - 1)), any_low = low_of(rq, query_of(rq, w.row0));
            w.from = max(static_cast<int32_t>(t0 + (j0 << a.span)), any_low & ~static_cast<int32_t>(kStep - 1));
            w.to = min(static_cast<int32_t>(min(t0 + (static_cast<uint64_t>(j1) << a.span), static_cast<uint64_t>(0x7FFFFFFF))), any_lim);
            return true;
        }
        return false;
    };

    // Page numbers through the scalar cache, a step ahead of the keys on them: a
    // vector load would have to be waited for together with the keys before it.
    const auto entry_of = [&](const Work &w, int32_t t) { return page_of(a, w.r, w.rq, static_cast<uint32_t>(t)); };
    const typename Tile<NB>::Places places(lane);
    const uint32_t page_bytes = a.cache.head_bytes * heads;
    const auto load = [&](Tile<NB> &to, const Work &w, int32_t t, uint32_t id0, uint32_t id1) {
        to.load(a.cache, a.cache.pages + w.h * a.cache.head_bytes, page_bytes, static_cast<uint32_t>(t), id0, id1, places);
    };

    Rows<NB, P> rows;
    typename Rows<NB, P>::Ahead ahead;
    Work w;
    bool says = false;  // this share has written its split
    int32_t t = 0;
    uint32_t id0 = 0, id1 = 0;  // of the step after this one, if it is the same tile's
    int32_t lim = 0, low = 0, any_lim = 0, any_low = 0, all_lim = 0, all_low = 0;
    bool mixed = false;
    const auto begin_tile = [&]() __attribute__((always_inline)) {
        const int32_t qa = query_of(w.rq, w.row0), qb = query_of(w.rq, w.row0 + w.count - 1);
        const int32_t mine_q = query_of(w.rq, w.row0 + min(lane & 15, w.count - 1));
        any_lim = lim_of(w.rq, qb), any_low = low_of(w.rq, qa), all_lim = lim_of(w.rq, qa), all_low = low_of(w.rq, qb);
        lim = lim_of(w.rq, mine_q), low = low_of(w.rq, mine_q);
        mixed = qa != qb;
        t = w.from;
        if (w.from < w.to) id0 = entry_of(w, t + kStep), id1 = entry_of(w, t + kStep + 16);
        rows.begin(a, ahead, w.rq, w.h, w.row0, w.count, lane);
    };
    // The keys in `now` are multiplied while those after them, of the same tile of
    // queries or the next, are on their way into `then`.  They are asked for in every
    // case (where there are none, some are again), so that it is known how many
    // loads are younger than the ones that are waited for.
    const auto advance = [&](const Tile<NB> &now, Tile<NB> &then) __attribute__((always_inline)) {
        const bool ends = t + static_cast<int32_t>(kStep) >= w.to;
        Work after = w;
        bool more = true;
        int32_t t_then = t + static_cast<int32_t>(kStep);
        uint32_t then0 = id0, then1 = id1;
        if (ends) {
            more = next(after);
            t_then = more && after.from < after.to ? after.from : 0;
            // without keys there may be no pages either
            then0 = then1 = 0xFFFFFFFFu;
            if (more && after.from < after.to) then0 = entry_of(after, t_then), then1 = entry_of(after, t_then + 16);
            if (more) Rows<NB, P>::ask(a, ahead, after.rq, after.h, after.row0, after.count, lane);
        } else {
            id0 = entry_of(w, t_then + kStep), id1 = entry_of(w, t_then + kStep + 16);
        }
        load(then, after, t_then, then0, then1);
        if (t < w.to)
            rows.step(a, now, static_cast<uint32_t>(t), lane,
                      t + static_cast<int32_t>(kStep) > all_lim || t < all_low || now.bad != 0, lim, low, any_lim, any_low, mixed);
        if (!ends) {
            t = t_then;
            return true;
        }
        const uint32_t g = lane >> 4, i = lane & 15, row = w.row0 + i;
        float sum = rows.sum + __shfl_xor(rows.sum, 16);
        sum += __shfl_xor(sum, 32);
        if (i < w.count) {
            const uint32_t query = static_cast<uint32_t>(query_of(w.rq, row));
            const uint64_t token = static_cast<uint64_t>(w.rq.first) + query;
            const uint32_t head = w.h * a.group + (row - query * a.group);
            float *part = a.parts + ((static_cast<uint64_t>(share) * 2 + (w.first ? 1 : 0)) * kTileRows + i) * part_row(NB);
#pragma unroll
            for (int e = 0; e < S::kLane / 2; ++e) {
                const uint32_t at = 4 * S::kLane * g + 8 * e;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = rows.o[(8 * e + k) % S::kLane][(8 * e + k) / S::kLane];
                if (w.whole) {
                    write_row(a, token, head, at, v, sum, rows.top);
                } else if (32 * NB == 16 * S::kLane || at < 32 * NB) {
                    __builtin_memcpy(__builtin_assume_aligned(part + at, 16), v, 32);
                }
            }
            if (!w.whole && g == 0) {
                part[32 * NB] = rows.top;
                part[32 * NB + 1] = sum;
            }
        }
        if (w.first && !w.whole) {
            says = true;
            if (lane == 0)  // up to the share that holds the tile's last unit
                a.splits[share] = {share_of(w.last) - share + 1, 2 * share + 1, 2 * share + 2, 2, w.h, w.row0, w.count,
                                   static_cast<uint32_t>(w.rq.first)};
        }
        if (more) {
            w = after;
            begin_tile();
        }
        return more;
    };
    if (next(w)) {
        Tile<NB> one, two;
        Rows<NB, P>::ask(a, ahead, w.rq, w.h, w.row0, w.count, lane);
        const bool any = w.from < w.to;
        load(one, w, any ? w.from : 0, any ? entry_of(w, w.from) : 0xFFFFFFFFu, any ? entry_of(w, w.from + 16) : 0xFFFFFFFFu);
        begin_tile();
        while (advance(one, two) && advance(two, one)) {
        }
    }
    if (!says && lane == 0) a.splits[share].parts = 0;
}

}  // namespace

template <int P>
void launch_kv4_few(const AttentionArgs &a, uint32_t waves, hipStream_t stream) {
    by_blocks(a.cache.blocks, [&](auto nb) {
        kv4_attention_kernel<decltype(nb)::value, P><<<(waves + kFewWaves - 1) / kFewWaves, kFewThreads, 0, stream>>>(a, waves);
    });
    BSQ_HIP(hipGetLastError());
}

}  // namespace bsq
