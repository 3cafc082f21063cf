// Attention over the paged MX4 cache: single tokens and a few queries a request
// (kv4_attention.hpp), the entry point, and the join of split tiles.
#include "kv4_attention.hpp"

#include <algorithm>
#include <cmath>

namespace bsq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kStep = 32;              // keys a wave takes at once
constexpr uint32_t kSpan = kStep * kWaves;  // keys a workgroup takes at once

// A tile's work: units of a.span keys (at least one, which writes the zeros of
// queries that see none), and kExtra more for what a tile costs beside its keys:
// page numbers, queries and first keys are waited for one after another, and the
// waves' sums are joined.
constexpr uint32_t kExtra = 2;

__device__ __forceinline__ uint32_t first_key(const AttentionArgs &a, const Request &q) {
    return a.window == 0 ? 0u : static_cast<uint32_t>(max(q.past() + 1 - static_cast<int64_t>(a.window), static_cast<int64_t>(0))) & ~(kStep - 1);
}
__device__ __forceinline__ uint32_t spans_of(const AttentionArgs &a, const Request &q) {
    const uint32_t first = first_key(a, q), length = static_cast<uint32_t>(q.length);
    return length > first ? (length - first + a.span - 1) / a.span : 1u;
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
    static constexpr int kRow = 16 * kLane + 4;  // floats of a row of sums in LDS
};

// 32 keys and values as a lane takes them.  Lane l = 16 g + i.  Keys: the row of
// token 16 a + 4 (i % 4) + i / 4 of the two sixteens a, channels [8 NB g, 8 NB (g
// + 1)).  The products' lane then holds, for query i, the tokens 16 a + 4 r + g =
// 4 j + g with j = 4 a + r: the eight that it holds of the values' rows, channels
// [kLane i, kLane (i + 1)), so the weights stay where they are.
template <int NB>
struct Tile {
    using S = Shape<NB>;
    uint32_t k[2][NB], ks[2][S::kScales], v[8][S::kWords], vs[2];
    uint32_t bad;  // bit a: the sixteen is on no page

    __device__ __forceinline__ void load(const AttentionArgs &a, uint32_t h, uint32_t t, uint32_t id0, uint32_t id1, uint32_t lane) {
        const uint32_t g = lane >> 4, i = lane & 15, page_mask = a.cache.page() - 1;
        const uint32_t row = a.cache.row_bytes();
        bad = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t id = s ? id1 : id0;
            if (id >= a.cache.count) {
                bad |= 1u << s;
                id = 0;
            }
            const uint8_t *head = a.cache.head(id, h);
            const uint32_t in = (t + 16 * s) & page_mask;
            const uint8_t *kp = head + a.cache.codes_at(0, in), *vp = head + a.cache.codes_at(1, in);
            const uint8_t *ksp = head + a.cache.scale_at(0, in, 0), *vsp = head + a.cache.scale_at(1, in, 0);
            const uint32_t token = 4 * (i & 3) + (i >> 2);
            __builtin_memcpy(k[s], __builtin_assume_aligned(kp + token * row + g * (4 * NB), NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), 4 * NB);
            const uint32_t ci = S::kLanes == 16 ? i : min(i, static_cast<uint32_t>(S::kLanes - 1));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint8_t *p = vp + (4 * r + g) * row + ci * (S::kLane / 2);
                if constexpr (S::kLane == 2) v[4 * s + r][0] = *p;
                else if constexpr (S::kLane == 4) v[4 * s + r][0] = *reinterpret_cast<const uint16_t *>(p);
                else __builtin_memcpy(v[4 * s + r], __builtin_assume_aligned(p, 4 * S::kWords), 4 * S::kWords);
            }
#pragma unroll
            for (int u = 0; u < S::kScales; ++u) {
                const uint32_t b = NB % 4 == 0 ? g * (NB / 4) + u : (g * NB + u) >> 2;
                ks[s][u] = ksp[(i >> 2) * (4 * NB) + 4 * b + (i & 3)];
            }
            vs[s] = *reinterpret_cast<const uint32_t *>(vsp + g * (4 * NB) + 4 * ((ci * S::kLane) >> 5));
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

    __device__ __forceinline__ void begin(const AttentionArgs &a, const Request &rq, uint32_t h, uint32_t row0, uint32_t rows, uint32_t lane) {
        const uint32_t g = lane >> 4, i = lane & 15, row = row0 + i;
        const uint64_t token = static_cast<uint32_t>(rq.first) + row / a.group;
        const uint64_t at = token * a.ldq + static_cast<uint64_t>(h * a.group + row % a.group) * a.cache.dim;
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            const uint32_t c = (g * NB + s) * 8;
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (i < rows && c < a.cache.dim)
                by_device_type(a.q_type, [&](auto t) { load8<decltype(t)::value>(a.q, at + c, a.cache.dim - c, x); });
            if (a.negate) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = -x[e];
            }
            u32x4 w[P];
            pieces<P>(x, w);
#pragma unroll
            for (int p = 0; p < P; ++p) q[p][s] = w[p];
        }
#pragma unroll
        for (int c = 0; c < S::kLane; ++c) o[c] = f32x4{0, 0, 0, 0};
        top = -__builtin_inff();
        base = sum = 0.0f;
    }

    // lim, low: the query sees the tokens [low, lim).  any_lim, any_low: some of
    // the tile's queries see those.
    template <bool MASKED>
    __device__ __forceinline__ void step(const AttentionArgs &a, const Tile<NB> &tile, uint32_t t, uint32_t lane, int32_t lim,
                                         int32_t low, int32_t any_lim, int32_t any_low, bool mixed) {
        const uint32_t g = lane >> 4, i = lane & 15;
        f32x4 x[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            x[s] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                const float scale = __uint_as_float(tile.ks[s][NB % 4 == 0 ? u / 4 : NB <= 2 ? 0 : u] << 23);
                const uint32_t w = tile.k[s][u];
                const u32x4 k = {cvt(w, scale, 0), cvt(w, scale, 1), cvt(w, scale, 2), cvt(w, scale, 3)};
#pragma unroll
                for (int p = 0; p < P; ++p) x[s] = mfma(k, q[p][u], x[s]);
            }
        }
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = x[j >> 2][j & 3] * a.factor;
            if constexpr (MASKED) {
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

        uint32_t v[8][S::kWords];
        float scale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t byte = (tile.vs[j >> 2] >> (8 * (j & 3))) & 0xFFu;
#pragma unroll
            for (int d = 0; d < S::kWords; ++d) v[j][d] = tile.v[j][d];
            if constexpr (MASKED) {
                // what no query sees may hold anything, NaN among it
                const int32_t at = static_cast<int32_t>(t + 4 * j + g);
                if (at >= any_lim || at < any_low || (tile.bad >> (j >> 2) & 1)) {
                    byte = 127;
#pragma unroll
                    for (int d = 0; d < S::kWords; ++d) v[j][d] = 0;
                }
                if (mixed) poison(a, byte, v[j], t + 4 * j, lane, lim, low);
            }
            scale[j] = __uint_as_float(byte << 23);
        }
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

// Each workgroup takes an equal share of all units of all requests' tiles: every
// tile of every head, in order, so that contexts of any lengths keep all CUs busy
// alike.  A tile whose keys lie in one share is written at once; of one whose do
// not, each share leaves its sums, and the join below adds them.
template <int NB, int P>
__global__ __launch_bounds__(kThreads, NB <= 4 ? 2 : 1) void kv4_attention_kernel(AttentionArgs a) {
    using S = Shape<NB>;
    __shared__ float tops[kWaves][kTileRows], totals[kWaves][kTileRows];
    __shared__ __attribute__((aligned(16))) float acc[kWaves][kTileRows][S::kRow];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t heads = a.cache.heads;

    // a lane's run of requests, and the units before it: every wave for itself,
    // without a barrier
    const uint32_t per = (a.requests + 63) / 64;
    const uint32_t r_begin = min(lane * per, a.requests), r_end = min(r_begin + per, a.requests);
    Request own{0, 0, 0};  // with one request a lane
    uint32_t mine = 0;
    for (uint32_t i = r_begin; i < r_end; ++i) {
        own = load_request(a, i);
        mine += tiles_of(a, own) * (spans_of(a, own) + kExtra);
    }
    mine *= heads;
    const uint32_t up_to = wave_prefix(mine), total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(up_to), 63));
    // no share is empty but those behind the last: a split tile's lie side by side
    const uint32_t shares = min(total, gridDim.x), share = blockIdx.x;
    if (share >= shares) {
        if (tid == 0) a.splits[share].parts = 0;
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
    uint32_t r = in_lane * per, base = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(up_to - mine), static_cast<int>(in_lane)));
    Request rq = request(r);
    bool says = false;  // this workgroup has written its split

    Rows<NB, P> rows;
    for (uint32_t x = begin; x < end;) {
        const uint32_t spans = spans_of(a, rq), units = spans + kExtra, tiles = tiles_of(a, rq);
        const uint32_t n = tiles * units * heads;
        if (x >= base + n) {
            if (++r >= a.requests) break;  // starts that overlap
            base += n;
            rq = request(r);
            continue;
        }
        const uint32_t tile = (x - base) / units, u0 = (x - base) - tile * units, u1 = min(units, u0 + (end - x));
        const uint32_t h = tile / tiles, row0 = (tile - h * tiles) * kTileRows;
        const uint32_t count = min(kTileRows, static_cast<uint32_t>(rq.count) * a.group - row0);
        x += u1 - u0;
        // the units ahead of the keys come first
        const uint32_t j0 = max(u0, kExtra) - kExtra, j1 = max(u1, kExtra) - kExtra;
        if (j1 <= j0) continue;

        // what the tile's queries see
        const int32_t qa = static_cast<int32_t>(row0 / a.group), qb = static_cast<int32_t>((row0 + count - 1) / a.group);
        const int32_t past = rq.past(), window = static_cast<int32_t>(min(a.window, 0x7FFFFFFFu));
        const auto lim_of = [&](int32_t query) { return a.causal ? past + query + 1 : rq.length; };
        const auto low_of = [&](int32_t query) { return window ? past + query + 1 - window : 0; };
        const int32_t any_lim = lim_of(qb), any_low = low_of(qa), all_lim = lim_of(qa), all_low = low_of(qb);
        const int32_t mine_q = static_cast<int32_t>((row0 + min(lane & 15, count - 1)) / a.group);
        const int32_t lim = lim_of(mine_q), low = low_of(mine_q);
        const uint32_t t0 = first_key(a, rq);
        const int32_t from = max(static_cast<int32_t>(t0 + j0 * a.span), any_low & ~static_cast<int32_t>(kStep - 1));
        const int32_t to = min(static_cast<int32_t>(min(t0 + static_cast<uint64_t>(j1) * a.span, static_cast<uint64_t>(0x7FFFFFFF))), any_lim);

        const int32_t t_first = from + static_cast<int32_t>(wave * kStep);
        const int32_t *entries = a.table + static_cast<uint64_t>(r) * a.width;
        const uint32_t last_entry = static_cast<uint32_t>(max(rq.length - 1, 0)) >> a.cache.shift;
        uint32_t ids = 0;
        // page numbers of 32 steps, a lane each sixteen
        const auto load = [&](Tile<NB> &tile_, int32_t t, uint32_t it) {
            if ((it & 31) == 0) {
                const uint32_t at = static_cast<uint32_t>(t) + (lane >> 1) * kSpan + (lane & 1) * 16;
                ids = static_cast<uint32_t>(entries[min(at >> a.cache.shift, last_entry)]);
            }
            const int from_lane = static_cast<int>((it & 31) * 2);
            tile_.load(a, h, static_cast<uint32_t>(t), static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ids), from_lane)),
                       static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ids), from_lane + 1)), lane);
        };
        const auto compute = [&](const Tile<NB> &tile_, int32_t t) {
            if (t + static_cast<int32_t>(kStep) <= all_lim && t >= all_low && tile_.bad == 0)
                rows.template step<false>(a, tile_, static_cast<uint32_t>(t), lane, lim, low, any_lim, any_low, false);
            else
                rows.template step<true>(a, tile_, static_cast<uint32_t>(t), lane, lim, low, any_lim, any_low, qa != qb);
        };
        Tile<NB> one, two;
        if (t_first < to) load(one, t_first, 0);
        rows.begin(a, rq, h, row0, count, lane);  // while the first keys are on their way
        if (t_first < to) {
            uint32_t it = 0;
            for (int32_t t = t_first; t < to; t += 2 * static_cast<int32_t>(kSpan)) {
                const int32_t second = t + static_cast<int32_t>(kSpan), third = second + static_cast<int32_t>(kSpan);
                if (second < to) load(two, second, it + 1);
                compute(one, t);
                if (second >= to) break;
                if (third < to) load(one, third, it + 2);
                compute(two, second);
                it += 2;
            }
        }

        // the waves' sums together
        float sum = rows.sum + __shfl_xor(rows.sum, 16);
        sum += __shfl_xor(sum, 32);
        const uint32_t g = lane >> 4, i = lane & 15;
        if (g == 0) {
            tops[wave][i] = rows.top;
            totals[wave][i] = sum;
        }
        if (i < count) {
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
                if (32 * NB == 16 * S::kLane || (4 * g + rr) * S::kLane < 32 * NB) {
                    float *p = &acc[wave][i][(4 * g + rr) * S::kLane];
#pragma unroll
                    for (int c = 0; c < S::kLane; ++c) p[c] = rows.o[c][rr];
                }
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == spans;
        float *part = a.parts + (static_cast<uint64_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * (kTileRows * part_row(NB));
        for (uint32_t item = tid; item < count * (4 * NB); item += kThreads) {
            const uint32_t n_row = item / (4 * NB), at = (item - n_row * (4 * NB)) * 8;
            float top = tops[0][n_row];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, tops[w][n_row]);
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, all = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                // without a reference there are zeros, or NaN
                const float keep = tops[w][n_row] == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(tops[w][n_row] - top);
                all += keep * totals[w][n_row];
                const float *p = &acc[w][n_row][at];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += keep * p[e];
            }
            if (whole) {
                const uint32_t row = row0 + n_row;
                write_row(a, static_cast<uint64_t>(rq.first) + row / a.group, h * a.group + row % a.group, at, v, all, top);
            } else {
                float *p = part + n_row * part_row(NB);
#pragma unroll
                for (int e = 0; e < 8; ++e) p[at + e] = v[e];
                if (at == 0) {
                    p[32 * NB] = top;
                    p[32 * NB + 1] = all;
                }
            }
        }
        if (j0 == 0 && j1 < spans) {
            says = true;
            if (tid == 0) {
                // up to the share that holds the tile's last unit
                const uint32_t parts = share_of(base + (tile + 1) * units - 1) - share + 1;
                a.splits[share] = {parts, 2 * share + 1, 2 * share + 2, 2, h, row0, count, static_cast<uint32_t>(rq.first)};
            }
        }
        __syncthreads();  // LDS is free again
    }
    if (!says && tid == 0) a.splits[blockIdx.x].parts = 0;
}

// A wave a row of a split tile.
template <int NB>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttentionArgs a, uint32_t part_rows) {
    const Split s = a.splits[blockIdx.x];
    const uint32_t n_row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (s.parts == 0 || n_row >= s.rows) return;
    const auto part = [&](uint32_t b) {
        const uint64_t number = b == 0 ? s.first : s.next + static_cast<uint64_t>(b - 1) * s.step;
        return a.parts + (number * part_rows + n_row) * part_row(NB);
    };
    float top = -__builtin_inff();
    for (uint32_t b = lane; b < s.parts; b += 64) top = fmaxf(top, part(b)[32 * NB]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    // lanes: parts beside one another, eight channels each
    constexpr uint32_t kEights = 4 * NB, kBeside = NB <= 1 ? 16 : NB == 2 ? 8 : NB <= 4 ? 4 : 2;
    const uint32_t e = lane % (64 / kBeside), beside = lane / (64 / kBeside);
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, all = 0.0f;
    if (e < kEights)
        for (uint32_t b = beside; b < s.parts; b += kBeside) {
            const float *p = part(b);
            const float mine = p[32 * NB];
            const float keep = mine == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mine - top);
            all += keep * p[32 * NB + 1];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += keep * p[e * 8 + i];
        }
#pragma unroll
    for (uint32_t d = 64 / kBeside; d < 64; d <<= 1) {
        all += __shfl_xor(all, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += __shfl_xor(v[i], d);
    }
    if (beside != 0 || e >= kEights) return;
    const uint32_t row = s.row0 + n_row;
    write_row(a, static_cast<uint64_t>(s.first_token) + row / a.group, s.head * a.group + row % a.group, e * 8, v, all, top);
}

// Requests of more rows than this are a prompt's: 16 rows a tile read and convert
// the keys once for each tile, 128 rows once for them all.
constexpr uint32_t kFewRows = 64;

struct Plan {
    uint32_t few;               // AttentionArgs' own
    uint32_t span = kSpan;      // AttentionArgs' own
    uint32_t groups = 0;        // of the kernel of few queries
    uint64_t tiles = 0;         // of the prompts' kernel
    uint32_t each = 1;
    uint64_t splits = 0, parts_bytes = 0, bytes = 0;
};
void check_sizes(const Kv4Cache &c, uint32_t width, uint32_t requests, uint64_t tokens, uint32_t q_heads) {
    BSQ_REQUIRE(q_heads >= 1 && q_heads % c.heads == 0, "kv4 attention: query heads are a multiple of the cache's");
    BSQ_REQUIRE(q_heads <= 65535, "kv4 attention: up to 65535 query heads");
    BSQ_REQUIRE(tokens <= 0x7FFFFFFFull && tokens * (q_heads / c.heads) <= 0x7FFFFFFFull, "kv4 attention: too many queries");
    BSQ_REQUIRE(requests <= 1u << 20, "kv4 attention: up to 2^20 requests");
    BSQ_REQUIRE(static_cast<uint64_t>(width) << c.shift <= 0x7FFFFFFFull - kSpan, "kv4 attention: rows of the table are too long");
}
Plan plan_of(const Kv4Cache &c, uint32_t width, uint32_t requests, uint64_t tokens, uint32_t most, uint32_t q_heads) {
    const uint64_t group = q_heads / c.heads, keys = std::max<uint64_t>(static_cast<uint64_t>(width) << c.shift, 1);
    const uint64_t rows = std::min<uint64_t>(tokens, static_cast<uint64_t>(requests) * most) * group;
    const uint64_t some = std::min<uint64_t>(requests, tokens);
    const bool prompts = static_cast<uint64_t>(most) * group > kFewRows;
    Plan p;
    // one request is one kernel's, whatever its queries
    p.few = prompts ? (requests == 1 ? 0 : kFewRows) : 0xFFFFFFFFu;
    uint64_t parts = 0;
    if (p.few > 0) {  // no more tiles and spans than these
        const uint64_t tiles = (rows / kTileRows + some) * c.heads;
        uint64_t units = ceil_div(keys, p.span) + 1 + kExtra;
        for (; tiles * units >= 1ull << 31 && p.span < 1u << 30; units = ceil_div(keys, p.span) + 1 + kExtra) p.span *= 2;
        BSQ_REQUIRE(tiles * units < 1ull << 31, "kv4 attention: too many queries");
        p.groups = static_cast<uint32_t>(std::min<uint64_t>(2ull * cu_count(), tiles * units));
        p.splits = p.groups;
        parts = static_cast<uint64_t>(p.groups) * 2 * kTileRows;
    }
    if (prompts) {
        p.tiles = rows / kPromptRows + std::min<uint64_t>(some, ceil_div(rows, p.few + 1));
        // two workgroups a CU; a share of at least 1024 keys
        const uint64_t shares = 2ull * cu_count() / (p.tiles * c.heads);
        p.each = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(shares, keys / 1024)));
        if (p.each > 1) {
            p.splits = std::max<uint64_t>(p.splits, p.tiles * c.heads);
            parts = std::max<uint64_t>(parts, p.tiles * c.heads * p.each * kPromptRows);
        }
    }
    p.parts_bytes = round256(parts * part_row(c.blocks) * 4);
    p.bytes = p.parts_bytes + round256(p.splits * sizeof(Split));
    return p;
}

template <int NB>
void join(const AttentionArgs &a, uint64_t splits, uint32_t part_rows, uint64_t rows, hipStream_t s) {
    rows = std::min<uint64_t>(rows, part_rows);
    kv4_join_kernel<NB><<<dim3(static_cast<unsigned>(splits), static_cast<unsigned>((rows + 3) / 4)), 256, 0, s>>>(a, part_rows);
    BSQ_HIP(hipGetLastError());
}

}  // namespace
}  // namespace bsq

using namespace bsq;

extern "C" {

uint64_t bsq_kv4_attention_workspace(const bsq_kv4_cache_t *cache, uint32_t width, uint32_t requests, uint64_t tokens,
                                     uint32_t most, uint32_t q_heads) {
    return size_query([&] {
        const Kv4Cache c = kv4_cache(cache, false);
        check_sizes(c, width, requests, tokens, q_heads);
        return plan_of(c, width, requests, tokens, most, q_heads).bytes;
    });
}

int bsq_kv4_attention(const bsq_kv4_cache_t *cache, const int32_t *d_table, uint32_t width, const int32_t *d_lengths,
                      const int32_t *d_starts, uint32_t requests, const void *d_q, int q_type, uint64_t tokens, uint32_t most,
                      uint32_t q_heads, uint64_t ldq, float scale, int causal, uint32_t window, void *d_out, int out_type,
                      uint64_t ldo, float *d_lse, void *d_work, uint64_t work_bytes, void *stream) {
    return entry([&] {
        const Mx4Type tq = type_of(q_type), to = type_of(out_type);
        const bool some = tokens > 0 && requests > 0 && most > 0;
        AttentionArgs a{};
        a.cache = kv4_cache(cache, some);
        check_sizes(a.cache, width, requests, tokens, q_heads);
        const uint64_t row = static_cast<uint64_t>(q_heads) * a.cache.dim;
        BSQ_REQUIRE(ldq >= row && ldo >= row, "kv4 attention: rows overlap");
        BSQ_REQUIRE(ldq <= 1ull << 28 && ldo <= 1ull << 28, "kv4 attention: rows too far apart");
        BSQ_REQUIRE(std::isfinite(scale), "kv4 attention: the scale is not finite");
        BSQ_REQUIRE(causal == 0 || causal == 1, "kv4 attention: causal is 0 or 1");
        BSQ_REQUIRE(causal == 1 || window == 0, "kv4 attention: a window is of causal attention");
        BSQ_REQUIRE(d_starts != nullptr || tokens == requests, "kv4 attention: without starts each request has one query");
        if (!some) return;
        BSQ_REQUIRE(d_lengths != nullptr && (width == 0 || d_table != nullptr), "kv4 attention: null argument");
        check_dense(d_q, tq, "kv4 attention: null queries");
        check_dense(d_out, to, "kv4 attention: null output");
        const Plan p = plan_of(a.cache, width, requests, tokens, most, q_heads);
        check_work(d_work, work_bytes, p.bytes);
        const int depth = std::max(tq == Mx4Type::F32 ? 3 : tq == Mx4Type::F16 ? 2 : 1, to == Mx4Type::F32 ? 3 : to == Mx4Type::F16 ? 2 : 1);
        a.table = d_table;
        a.lengths = d_lengths;
        a.starts = d_starts;
        a.width = width;
        a.requests = requests;
        a.q = static_cast<const uint8_t *>(d_q);
        a.q_type = tq;
        a.out_type = to;
        a.ldq = ldq;
        a.ldo = ldo;
        a.tokens = static_cast<uint32_t>(tokens);
        a.most = std::min<uint32_t>(most, 0x7FFFFFFFu);
        a.group = q_heads / a.cache.heads;
        a.factor = static_cast<float>(std::fabs(static_cast<double>(scale)) * 1.44269504088896340736);
        a.negate = scale < 0.0f;
        a.causal = causal != 0;
        a.window = window;
        a.out = static_cast<uint8_t *>(d_out);
        a.lse = d_lse;
        a.parts = static_cast<float *>(d_work);
        a.splits = reinterpret_cast<Split *>(static_cast<uint8_t *>(d_work) + p.parts_bytes);
        a.few = p.few;
        a.span = p.span;
        a.each = p.each;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const uint64_t rows = static_cast<uint64_t>(a.most) * a.group;
        by_blocks(a.cache.blocks, [&](auto nb) {
            constexpr int NB = decltype(nb)::value;
            if (p.groups > 0) {
                if (depth == 1) kv4_attention_kernel<NB, 1><<<p.groups, kThreads, 0, s>>>(a);
                else if (depth == 2) kv4_attention_kernel<NB, 2><<<p.groups, kThreads, 0, s>>>(a);
                else kv4_attention_kernel<NB, 3><<<p.groups, kThreads, 0, s>>>(a);
                BSQ_HIP(hipGetLastError());
                if (p.groups > 1) join<NB>(a, p.groups, kTileRows, rows, s);
            }
            if (p.tiles > 0) {
                launch_kv4_prompt(a, depth, p.tiles, s);
                if (p.each > 1) join<NB>(a, p.tiles * a.cache.heads, kPromptRows, rows, s);
            }
        });
    });
}

}  // extern "C"
