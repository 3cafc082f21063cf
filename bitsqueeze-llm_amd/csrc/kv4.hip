// A step's bookkeeping, rotary positions, and the way into and out of the paged
// MX4 cache (kv4.hpp).
#include "kv4.hpp"

#include <algorithm>
#include <cmath>

namespace bsq {
namespace {

// ---------------------------------------------------------------------------
// the plan of a step
// ---------------------------------------------------------------------------
// Everything hangs on prefix sums over the requests: of the pages that the ended
// ones give back, and of the tokens and pages that the others take.  One workgroup
// forms them all at once, a run of requests a thread; the places of the tokens then
// need only a search in the starts.  Small steps do both in the one launch, as a
// second costs more than the search; large ones spread the places over a grid.
// What bounds it are waits one after another: lengths, the sums' exchange between
// waves, the ended requests' rows, the pages of new tokens (64 requests 7.7 us, the
// host's launch; 2000 with 40 that end 20 us).
constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanMostRequests = 16384;
constexpr uint32_t kPlanOneLaunch = 4096;  // places

struct PlanArgs {
    const int32_t *lengths, *more;
    uint32_t requests;
    int32_t *table;
    uint32_t width, shift;
    int32_t *free;
    uint32_t pages;
    const int32_t *count;
    int32_t *lengths_out, *left, *starts;
    uint32_t tokens;
    int32_t *of, *positions, *slots;
    int32_t *first;  // requests + 1: the first page of each from the stack's top, -1 if not served; the top
};

// Three sums over the threads before this one, and over all.
struct PlanSums {
    uint64_t v[3];
};
__device__ __forceinline__ PlanSums plan_prefix(const PlanSums mine, PlanSums *of_waves, PlanSums &all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    PlanSums up = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        PlanSums o;
#pragma unroll
        for (int i = 0; i < 3; ++i) o.v[i] = __shfl_up(up.v[i], d);
#pragma unroll
        for (int i = 0; i < 3; ++i) up.v[i] += lane >= static_cast<uint32_t>(d) ? o.v[i] : 0;
    }
    if (lane == 63) of_waves[wave] = up;
    __syncthreads();
    all = {};
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
        const PlanSums s = of_waves[w];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            up.v[i] += w < wave ? s.v[i] : 0;
            all.v[i] += s.v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) up.v[i] -= mine.v[i];
    return up;
}

struct PlanRequest {
    int64_t past, more;
    uint32_t held, need;
    bool ended, wide;
};
__device__ __forceinline__ PlanRequest plan_request(const PlanArgs &a, uint32_t r) {
    PlanRequest q;
    q.past = max(a.lengths[r], 0);
    const int32_t n = a.more[r];
    q.ended = n < 0;
    q.more = max(n, 0);
    const int64_t page = 1ll << a.shift, room = static_cast<int64_t>(a.width) << a.shift;
    q.wide = !q.ended && q.past + q.more > room;
    q.held = static_cast<uint32_t>((min(q.past, room) + page - 1) >> a.shift);
    q.need = q.ended || q.wide ? 0u : static_cast<uint32_t>((q.past + q.more + page - 1) >> a.shift) - q.held;
    return q;
}

// The last r with starts[r] <= t.
__device__ __forceinline__ uint32_t plan_search(const int32_t *starts, uint32_t requests, int32_t t) {
    uint32_t lo = 0, hi = requests;  // starts[lo] <= t < starts[hi], if any
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void plan_place(const PlanArgs &a, uint32_t t, const int32_t *starts, int32_t total, uint32_t top) {
    int32_t of = -1, position = -1, slot = -1;
    if (static_cast<int32_t>(t) < total) {
        const uint32_t r = plan_search(starts, a.requests, static_cast<int32_t>(t));
        of = static_cast<int32_t>(r);
        const int32_t first = a.first[r];
        if (first >= 0) {
            const int32_t n = starts[r + 1] - starts[r], past = a.lengths_out[r] - n;
            const uint32_t page = 1u << a.shift, held = (static_cast<uint32_t>(past) + page - 1) >> a.shift;
            position = past + static_cast<int32_t>(t) - starts[r];
            const uint32_t place = static_cast<uint32_t>(position) >> a.shift, in = static_cast<uint32_t>(position) & (page - 1);
            int32_t *entry = a.table + static_cast<uint64_t>(r) * a.width + place;
            int32_t number;
            if (place < held) {
                number = *entry;
            } else {
                number = a.free[top - 1 - (static_cast<uint32_t>(first) + place - held)];
                if (in == 0) *entry = number;  // a page's first token is new where the page is
            }
            if (static_cast<uint32_t>(number) < a.pages) slot = (number << a.shift) + static_cast<int32_t>(in);
        }
    }
    if (a.of != nullptr) a.of[t] = of;
    a.positions[t] = position;
    a.slots[t] = slot;
}

// ALL: the places too.
template <bool ALL>
__global__ __launch_bounds__(kPlanThreads) void kv4_plan_kernel(PlanArgs a) {
    struct Ended {
        uint32_t request, before, pages;
    };
    __shared__ PlanSums of_waves[kPlanThreads / 64];
    __shared__ Ended ended[kPlanThreads];
    __shared__ int32_t starts[ALL ? kPlanThreads + 1 : 1];
    __shared__ uint32_t taken[kPlanThreads / 64], unserved[kPlanThreads / 64];
    const uint32_t tid = threadIdx.x;
    const uint32_t count = min(static_cast<uint32_t>(max(*a.count, 0)), a.pages);
    const uint32_t per = (a.requests + kPlanThreads - 1) / kPlanThreads;
    const uint32_t r_begin = min(tid * per, a.requests), r_end = min(r_begin + per, a.requests);
    PlanSums mine{};
    for (uint32_t r = r_begin; r < r_end; ++r) {
        const PlanRequest q = plan_request(a, r);
        mine.v[0] += q.ended ? (1ull << 40) + q.held : 0;  // requests above, pages below
        mine.v[1] += static_cast<uint64_t>(q.more);
        mine.v[2] += q.need;
    }
    PlanSums all;
    PlanSums before = plan_prefix(mine, of_waves, all);
    constexpr uint64_t kLow = (1ull << 40) - 1;
    const uint32_t top = static_cast<uint32_t>(min(count + (all.v[0] & kLow), static_cast<uint64_t>(a.pages)));
    const uint32_t ends = static_cast<uint32_t>(all.v[0] >> 40);
    uint32_t most = 0, left_out = 0;
    {
        PlanSums at = before;
        for (uint32_t r = r_begin; r < r_end; ++r) {
            const PlanRequest q = plan_request(a, r);
            at.v[1] += static_cast<uint64_t>(q.more);
            at.v[2] += q.need;
            const bool fits = !q.wide && at.v[1] <= a.tokens && (q.need == 0 || at.v[2] <= top);
            const int32_t start = static_cast<int32_t>(min(at.v[1], static_cast<uint64_t>(a.tokens)));
            a.starts[r + 1] = start;
            if (ALL) starts[r + 1] = start;
            a.first[r] = q.ended || !fits ? -1 : q.need == 0 ? 0 : static_cast<int32_t>(at.v[2] - q.need);
            a.lengths_out[r] = q.ended ? 0 : static_cast<int32_t>(fits ? q.past + q.more : q.past);
            // the pages that are taken end with the last request that is served
            if (!q.ended && fits && q.need > 0) most = static_cast<uint32_t>(at.v[2]);
            if (!q.ended && !fits) ++left_out;
            // more of them than the list holds: a thread each below
            if (q.ended) {
                const uint64_t n = at.v[0] >> 40;
                const Ended e{r, static_cast<uint32_t>(at.v[0] & kLow), q.held};
                if (ends <= kPlanThreads) {
                    ended[n] = e;
                } else {
                    for (uint32_t i = 0; i < e.pages && count + static_cast<uint64_t>(e.before) + i < a.pages; ++i)
                        a.free[count + e.before + i] = a.table[static_cast<uint64_t>(r) * a.width + i];
                }
                at.v[0] += (1ull << 40) + q.held;
            }
        }
    }
    // what of the stack is taken, and how many requests are not served
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
        left_out += static_cast<uint32_t>(__shfl_xor(static_cast<int>(left_out), d));
    }
    if ((tid & 63) == 0) taken[tid >> 6] = most, unserved[tid >> 6] = left_out;
    __syncthreads();
    // the ended requests' pages, a wave a request
    if (ends <= kPlanThreads)
        for (uint32_t e = tid >> 6; e < ends; e += kPlanThreads / 64) {
            const Ended of = ended[e];
            const int32_t *from = a.table + static_cast<uint64_t>(of.request) * a.width;
            const uint64_t to = static_cast<uint64_t>(count) + of.before;
#pragma unroll 8
            for (uint32_t i = tid & 63; i < of.pages; i += 64)
                if (to + i < a.pages) a.free[to + i] = from[i];
        }
    if (tid == 0) {
        uint32_t all_taken = 0, all_unserved = 0;
#pragma unroll
        for (uint32_t w = 0; w < kPlanThreads / 64; ++w) all_taken = max(all_taken, taken[w]), all_unserved += unserved[w];
        a.starts[0] = 0;
        if (ALL) starts[0] = 0;
        a.first[a.requests] = static_cast<int32_t>(top);
        a.left[0] = static_cast<int32_t>(top - all_taken);
        a.left[1] = static_cast<int32_t>(all_unserved);
    }
    if constexpr (ALL) {
        __syncthreads();
        const int32_t total = static_cast<int32_t>(min(all.v[1], static_cast<uint64_t>(a.tokens)));
        for (uint32_t t = tid; t < a.tokens; t += kPlanThreads) plan_place(a, t, starts, total, top);
    }
}

constexpr uint32_t kPlaceThreads = 256;
__global__ __launch_bounds__(kPlaceThreads) void kv4_places_kernel(PlanArgs a) {
    extern __shared__ int32_t all_starts[];
    for (uint32_t r = threadIdx.x; r <= a.requests; r += kPlaceThreads) all_starts[r] = a.starts[r];
    __syncthreads();
    const uint32_t top = static_cast<uint32_t>(a.first[a.requests]);
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kPlaceThreads + threadIdx.x; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kPlaceThreads)
        plan_place(a, static_cast<uint32_t>(t), all_starts, all_starts[a.requests], top);
}

// ---------------------------------------------------------------------------
// rotary positions, append
// ---------------------------------------------------------------------------
// Angles grow with the position: at 10^6 radians FP32 is off by 0.06.  They are
// FP64 products, brought into [-pi/4, pi/4] with pi/2 in two parts, and sine and
// cosine their Taylor sums there (remainders below 2^-60); a token's serve all its
// heads.  A pair's products are FP64 for FP32 values, and for keys on their way into
// the cache: next to a border of its 4-bit codes a key falls on the side that the
// exact value is on.  Of 16-bit values they are FP32, a small part of the rounding
// that follows: 8192 tokens of 32 heads of 128, half of it turned, forward and
// gradient, take 57 us so, and 66 in FP64, whose conversions are slow.
__device__ __forceinline__ void sine_cosine(double t, double &s, double &c) {
    const double n = rint(t * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, t);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double x = r * r;
    double p = 1.0 / 355687428096000.0, q = 1.0 / 20922789888000.0;
    p = fma(p, x, -1.0 / 1307674368000.0);
    p = fma(p, x, 1.0 / 6227020800.0);
    p = fma(p, x, -1.0 / 39916800.0);
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, -1.0 / 5040.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, -1.0 / 6.0);
    const double sine = fma(p * x, r, r);
    q = fma(q, x, -1.0 / 87178291200.0);
    q = fma(q, x, 1.0 / 479001600.0);
    q = fma(q, x, -1.0 / 3628800.0);
    q = fma(q, x, 1.0 / 40320.0);
    q = fma(q, x, -1.0 / 720.0);
    q = fma(q, x, 1.0 / 24.0);
    q = fma(q, x, -0.5);
    const double cosine = fma(q, x, 1.0);
    const int quarter = static_cast<int>(static_cast<long long>(n)) & 3;
    s = quarter & 1 ? cosine : sine;
    c = quarter & 1 ? sine : cosine;
    if (quarter & 2) s = -s;
    if (quarter == 1 || quarter == 2) c = -c;
}

// i / d and the rest for i, d < 2^24, from 1 / d in FP32: at most one off, which is
// put right.  The compiler's division takes some 40 instructions.
struct Divisor {
    uint32_t d = 1;
    float inverse = 1.0f;
    Divisor() = default;
    explicit Divisor(uint32_t divisor) : d(divisor), inverse(1.0f / static_cast<float>(divisor)) {}
    __device__ __forceinline__ void operator()(uint32_t i, uint32_t &q, uint32_t &r) const {
        q = static_cast<uint32_t>(static_cast<float>(i) * inverse);
        r = i - q * d;
        if (static_cast<int32_t>(r) < 0) r += d, --q;
        else if (r >= d) r -= d, ++q;
    }
};

struct Turn {
    const double *frequencies = nullptr;  // none: nothing turns
    uint32_t half = 0;                    // pairs
    int interleaved = 0;
    double cosine = 1.0, sine = 1.0;  // factors
};

struct RowsArgs {
    Turn turn;
    const int32_t *positions, *slots;
    uint64_t tokens;
    uint32_t dim, per;  // tokens of a workgroup
    const uint8_t *q, *k, *v;
    uint8_t *qo;
    uint64_t ldq, ldqo, ldk, ldv;
    uint32_t q_heads;
    uint32_t chunks, rest;  // eights of pairs in a head, and of values that do not turn
    bool in_place;
    Kv4Cache cache;
    Divisor by_half, by_q_heads, by_chunks, by_rest, by_heads, by_key_eights, by_eights;
};

constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kRowTokens = 4;          // most of a workgroup
constexpr uint32_t kRowPairs = kKv4MaxDim / 2;
constexpr uint32_t kKeyBytes = 16384;       // turned keys held at once

// Eight pairs of a row, chunk c of the turning part; or eight values of the rest.
template <Mx4Type T>
struct Pairs {
    static constexpr int kWords = Eight<T>::kWords;
    float a[8], b[8];
    // as stored: loaded ahead of their use
    struct Words {
        Eight<T> a, b;
    };
    __device__ __forceinline__ static void load(Words &w, const uint8_t *row, const Turn &t, uint32_t c) {
        if (t.interleaved) {
            w.a.load(row, 16 * c, 2 * t.half);
            w.b.load(row, 16 * c + 8, 2 * t.half);
        } else {
            w.a.load(row, 8 * c, t.half);
            w.b.load(row + t.half * (T == Mx4Type::F32 ? 4 : 2), 8 * c, t.half);
        }
    }
    __device__ __forceinline__ static void values(const Eight<T> &e, float v[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (T == Mx4Type::F32) {
                v[i] = __uint_as_float(e.w[i]);
            } else {
                const uint32_t x = (e.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
                v[i] = T == Mx4Type::BF16 ? bf16_value(x) : f16_value(x);
            }
        }
    }
    // values [at, at + 8) of a row of n, as they are
    __device__ __forceinline__ static void move(const Eight<T> &e, uint8_t *row, uint32_t at, uint32_t n) {
        if (at + 8 <= n) {
            __builtin_memcpy(row + at * (T == Mx4Type::F32 ? 4 : 2), e.w, sizeof(e.w));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (at + i >= n) continue;
                if constexpr (T == Mx4Type::F32) reinterpret_cast<uint32_t *>(row)[at + i] = e.w[i];
                else reinterpret_cast<uint16_t *>(row)[at + i] = static_cast<uint16_t>(e.w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
    __device__ __forceinline__ explicit Pairs(const Words &w) {
        values(w.a, a);
        values(w.b, b);
    }
    __device__ __forceinline__ static void turn_one(float &x, float &y, const double2 u) {
        const double p = x, q = y;
        x = static_cast<float>(fma(p, u.x, -(q * u.y)));
        y = static_cast<float>(fma(q, u.x, p * u.y));
    }
    __device__ __forceinline__ static void turn_one(float &x, float &y, const float2 u) {
        const float p = x, q = y;
        x = fmaf(p, u.x, -(q * u.y));
        y = fmaf(q, u.x, p * u.y);
    }
    // cs: cosine and sine of pair i at cs[i * step]
    template <class Two>
    __device__ __forceinline__ void turn(const Turn &t, const Two *cs, uint32_t step) {
        if (t.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) turn_one(a[2 * i], a[2 * i + 1], cs[i * step]);
#pragma unroll
            for (int i = 0; i < 4; ++i) turn_one(b[2 * i], b[2 * i + 1], cs[(4 + i) * step]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn_one(a[i], b[i], cs[i * step]);
        }
    }
    __device__ __forceinline__ void store(uint8_t *row, const Turn &t, uint32_t c) const {
        const uint32_t at = 8 * c, left = t.half - at;
        if (t.interleaved) {
            store8<T>(row, 2 * at, 2 * left, a);
            store8<T>(row, 2 * at + 8, left > 4 ? 2 * left - 8 : 0, b);
        } else {
            store8<T>(row, at, left, a);
            store8<T>(row, t.half + at, left, b);
        }
    }
};

template <Mx4Type T>
__device__ __forceinline__ void pack(const RowsArgs &a, const Eight<T> &v, uint32_t which, uint32_t slot, uint32_t h, uint32_t c) {
    const uint32_t byte = mx4_scale_byte(f32_bits<T>(quad_max(v.top())));
    if (slot >> a.cache.shift >= a.cache.count) return;
    uint8_t *to = a.cache.head(slot >> a.cache.shift, h);
    const uint32_t t = slot & (a.cache.page() - 1);
    const uint32_t codes = byte == 255u ? 0u : v.codes(mx4_power(byte));
    *reinterpret_cast<uint32_t *>(to + a.cache.codes_at(which, t) + 4 * c) = codes;
    if ((c & 3) == 0) to[a.cache.scale_at(which, t, c >> 2)] = static_cast<uint8_t>(byte);
}

// A workgroup takes `per` tokens and of them the queries or the keys and values:
// eight of the one, eight of the other in turn, so that every XCD has both at once,
// queries that wait for memory and keys that compute.  Sines and cosines go through LDS, once a token; turned
// keys too, in their own type, since a pair's halves belong to two blocks.  A
// thread's words are on their way while sines are computed, and then one item
// ahead.  !KV: queries only, 29 us for 8192 tokens of 32 heads of 128 in BF16, 4.6
// TB/s.  With 8 heads of keys and values 48 us, 3.7 TB/s: packing them takes vector
// instructions and two barriers.
template <Mx4Type T, bool KV>
__global__ __launch_bounds__(kRowThreads) void kv4_rows_kernel(RowsArgs a) {
    constexpr uint32_t size = T == Mx4Type::F32 ? 4 : 2;
    using P = Pairs<T>;
    __shared__ double2 cs[kRowTokens * kRowPairs];
    float2 *cs32 = reinterpret_cast<float2 *>(cs);
    constexpr bool kWide = T == Mx4Type::F32;
    __shared__ __attribute__((aligned(16))) uint8_t turned[KV ? kKeyBytes : 16];
    const uint32_t tid = threadIdx.x;
    const uint32_t group = KV ? blockIdx.x / 16 * 8 + blockIdx.x % 8 : blockIdx.x;
    const uint64_t t0 = static_cast<uint64_t>(group) * a.per;
    if (KV && t0 >= a.tokens) return;
    const uint32_t here = static_cast<uint32_t>(min(static_cast<uint64_t>(a.per), a.tokens - t0));
    const Turn &turn = a.turn;
    const uint32_t chunks = a.chunks;
    const auto absent = [&](uint32_t t) { return a.positions != nullptr && a.positions[t0 + t] < 0; };
    const auto sines = [&](auto wide) {
        if (turn.frequencies == nullptr) return;
        for (uint32_t i = tid; i < here * turn.half; i += kRowThreads) {
            uint32_t t, j;
            a.by_half(i, t, j);
            double s, c;
            sine_cosine(static_cast<double>(a.positions[t0 + t]) * turn.frequencies[j], s, c);
            c *= turn.cosine, s *= turn.sine;
            const uint32_t to = (t * 8 + (j & 7)) * chunks + (j >> 3);
            if constexpr (decltype(wide)::value) cs[to] = {c, s};
            else cs32[to] = {static_cast<float>(c), static_cast<float>(s)};
        }
        __syncthreads();
    };
    if (!KV || blockIdx.x / 8 % 2 == 0) {
        if (a.q == nullptr) return;
        // what turns comes first, what is only moved behind it: waves do the one or the
        // other
        const uint32_t turning = here * a.q_heads * chunks, all = turning + (a.in_place ? 0u : here * a.q_heads * a.rest);
        struct Item {
            uint32_t t, h, c;
        };
        const auto item_of = [&](uint32_t i) {
            Item n;
            uint32_t row;
            if (i < turning) a.by_chunks(i, row, n.c);
            else a.by_rest(i - turning, row, n.c);
            a.by_q_heads(row, n.t, n.h);
            return n;
        };
        const auto load = [&](typename P::Words &w, uint32_t i, const Item &n) {
            const uint8_t *from = a.q + ((t0 + n.t) * a.ldq + static_cast<uint64_t>(n.h) * a.dim) * size;
            if (i < turning) P::load(w, from, turn, n.c);
            else w.a.load(from, 2 * turn.half + 8 * n.c, a.dim);
        };
        typename P::Words next;
        Item then{0, 0, 0};
        if (tid < all) load(next, tid, then = item_of(tid));
        sines(std::bool_constant<kWide>{});
        for (uint32_t i = tid; i < all; i += kRowThreads) {
            const typename P::Words now = next;
            const Item n = then;
            if (i + kRowThreads < all) load(next, i + kRowThreads, then = item_of(i + kRowThreads));
            if (absent(n.t)) continue;
            uint8_t *to = a.qo + ((t0 + n.t) * a.ldqo + static_cast<uint64_t>(n.h) * a.dim) * size;
            if (i < turning) {
                P p(now);
                if constexpr (kWide) p.turn(turn, cs + n.t * 8 * chunks + n.c, chunks);
                else p.turn(turn, cs32 + n.t * 8 * chunks + n.c, chunks);
                p.store(to, turn, n.c);
            } else {
                P::move(now.a, to, 2 * turn.half + 8 * n.c, a.dim);
            }
        }
        return;
    }
    if constexpr (KV) {
        const uint32_t eights = a.cache.blocks * 4, heads = a.cache.heads, rows = here * heads;
        const auto slot_of = [&](uint32_t t) { return absent(t) ? 0xFFFFFFFFu : static_cast<uint32_t>(a.slots[t0 + t]); };
        const uint32_t stride = a.cache.blocks * 32 * size + 16, most = kKeyBytes / stride, each = chunks + a.rest;
        const auto load_key = [&](typename P::Words &w, uint32_t r0, uint32_t i) {
            uint32_t n, c, t, h;
            a.by_key_eights(i, n, c);
            a.by_heads(r0 + n, t, h);
            const uint8_t *from = a.k + ((t0 + t) * a.ldk + static_cast<uint64_t>(h) * a.dim) * size;
            if (c < chunks) P::load(w, from, turn, c);
            else w.a.load(from, 2 * turn.half + 8 * (c - chunks), a.dim);
        };
        const bool turns = turn.frequencies != nullptr;
        typename P::Words next;
        if (turns && tid < min(most, rows) * each) load_key(next, 0, tid);
        // values; a quad of lanes never parts: `eights` is a multiple of four
        Eight<T> word;
        const auto value_at = [&](uint32_t i, uint32_t &t, uint32_t &h, uint32_t &c) {
            uint32_t row;
            a.by_eights(i, row, c);
            a.by_heads(row, t, h);
        };
        const auto load_value = [&](const uint8_t *base, uint64_t ld, uint32_t i) {
            uint32_t t, h, c;
            value_at(i, t, h, c);
            word.load(base + ((t0 + t) * ld + static_cast<uint64_t>(h) * a.dim) * size, 8 * c, a.dim);
        };
        const auto pack_rows = [&](const uint8_t *base, uint64_t ld, uint32_t which) {
            for (uint32_t i = tid; i < rows * eights; i += kRowThreads) {
                const Eight<T> now = word;
                if (i + kRowThreads < rows * eights) load_value(base, ld, i + kRowThreads);
                uint32_t t, h, c;
                value_at(i, t, h, c);
                pack<T>(a, now, which, slot_of(t), h, c);
            }
        };
        if (tid < rows * eights) load_value(a.v, a.ldv, tid);
        sines(std::true_type{});
        pack_rows(a.v, a.ldv, 1);
        if (!turns) {
            if (tid < rows * eights) load_value(a.k, a.ldk, tid);
            pack_rows(a.k, a.ldk, 0);
            return;
        }
        for (uint32_t r0 = 0; r0 < rows; r0 += most) {
            const uint32_t count = min(most, rows - r0);
            if (r0 > 0 && tid < count * each) load_key(next, r0, tid);
            for (uint32_t i = tid; i < count * each; i += kRowThreads) {
                const typename P::Words now = next;
                if (i + kRowThreads < count * each) load_key(next, r0, i + kRowThreads);
                uint32_t n, c, t, h;
                a.by_key_eights(i, n, c);
                a.by_heads(r0 + n, t, h);
                uint8_t *to = turned + n * stride;
                if (c < chunks) {
                    P p(now);
                    p.turn(turn, cs + t * 8 * chunks + c, chunks);
                    p.store(to, turn, c);
                } else {
                    P::move(now.a, to, 2 * turn.half + 8 * (c - chunks), a.dim);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < count * eights; i += kRowThreads) {
                uint32_t n, c, t, h;
                a.by_eights(i, n, c);
                a.by_heads(r0 + n, t, h);
                Eight<T> v;
                v.load(turned + n * stride, 8 * c, a.dim);
                pack<T>(a, v, 0, slot_of(t), h, c);
            }
            __syncthreads();
        }
    }
}

void launch_rows(const RowsArgs &rows, Mx4Type type, bool kv, hipStream_t stream) {
    RowsArgs a = rows;
    a.chunks = (a.turn.half + 7) / 8;
    a.rest = (a.dim - 2 * a.turn.half + 7) / 8;
    a.by_half = Divisor(std::max(a.turn.half, 1u));
    a.by_q_heads = Divisor(std::max(a.q_heads, 1u));
    a.by_chunks = Divisor(std::max(a.chunks, 1u));
    a.by_rest = Divisor(std::max(a.rest, 1u));
    a.by_key_eights = Divisor(std::max(a.chunks + a.rest, 1u));
    a.by_heads = Divisor(std::max(kv ? a.cache.heads : 1u, 1u));
    a.by_eights = Divisor(std::max(kv ? a.cache.blocks * 4 : 1u, 1u));
    // several tokens a workgroup share the wait for their sines, as long as three times
    // as many groups of tokens as CUs remain (with keys and values a group is two
    // workgroups)
    a.per = 1;
    while (a.per < kRowTokens && a.tokens / (2 * a.per) >= 3ull * cu_count()) a.per *= 2;
    static_assert(kRowTokens * 65535 * (kKv4MaxDim / 8 + 1) < 1u << 24, "items are divided in 24 bits");
    const uint64_t groups = ceil_div(a.tokens, a.per);
    BSQ_REQUIRE(groups <= 0xFFFFFFFFull / (2 * kRowThreads) - 16, "kv4: too many tokens");
    by_type(type, [&](auto ty) {
        const unsigned grid = static_cast<unsigned>(kv ? ceil_div(groups, 8) * 16 : groups);
        if (kv) kv4_rows_kernel<decltype(ty)::value, true><<<grid, kRowThreads, 0, stream>>>(a);
        else kv4_rows_kernel<decltype(ty)::value, false><<<grid, kRowThreads, 0, stream>>>(a);
    });
    BSQ_HIP(hipGetLastError());
}

// Eight values a lane; a workgroup takes `per` tokens.
template <Mx4Type T>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Cache cache, const int32_t *slots, uint64_t tokens, uint32_t per,
                                                       Divisor by_heads, Divisor by_eights, uint8_t *k, uint64_t ldk, uint8_t *v,
                                                       uint64_t ldv) {
    constexpr uint32_t size = T == Mx4Type::F32 ? 4 : 2;
    const uint32_t which = k == nullptr ? 1 : blockIdx.y;
    uint8_t *out = which ? v : k;
    const uint64_t ld = which ? ldv : ldk, t0 = static_cast<uint64_t>(blockIdx.x) * per;
    const uint32_t here = static_cast<uint32_t>(min(static_cast<uint64_t>(per), tokens - t0));
    for (uint32_t i = threadIdx.x; i < here * by_heads.d * by_eights.d; i += 256) {
        uint32_t row, c, t, h;
        by_eights(i, row, c);
        by_heads(row, t, h);
        const uint32_t slot = static_cast<uint32_t>(slots[t0 + t]), in = slot & (cache.page() - 1);
        if (slot >> cache.shift >= cache.count) continue;
        const uint8_t *from = cache.head(slot >> cache.shift, h);
        const uint32_t codes = *reinterpret_cast<const uint32_t *>(from + cache.codes_at(which, in) + 4 * c);
        const uint32_t byte = from[cache.scale_at(which, in, c >> 2)];
        const float scale = byte == 255u ? __builtin_nanf("") : byte == 0u ? 0x1p-127f : mx4_power(byte);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t n = (codes >> (4 * j)) & 15u;
            // E2M1: m / 2 at exponent 0, (1 + m / 2) 2^(e - 1) above; an FP32 with these bits,
            // times 2^126
            const float level = __uint_as_float((n & 7u) << 22) * 0x1p126f;
            x[j] = (n & 8u ? -level : level) * scale;
        }
        store8<T>(out + ((t0 + t) * ld + static_cast<uint64_t>(h) * cache.dim) * size, 8 * c, cache.dim - 8 * c, x);
    }
}

Turn turn_of(const bsq_rope_t *rope, uint32_t dim, int back) {
    BSQ_REQUIRE(rope->d_frequencies != nullptr, "rope: null frequencies");
    BSQ_REQUIRE((reinterpret_cast<uintptr_t>(rope->d_frequencies) & 7) == 0, "rope: frequencies unaligned");
    BSQ_REQUIRE(rope->dims >= 2 && rope->dims % 2 == 0 && rope->dims <= dim, "rope: an even number of dims, 2 to the head's");
    BSQ_REQUIRE(rope->interleaved == 0 || rope->interleaved == 1, "rope: interleaved is 0 or 1");
    BSQ_REQUIRE(std::isfinite(rope->factor), "rope: the factor is not finite");
    return {rope->d_frequencies, rope->dims / 2, rope->interleaved, rope->factor,
            back ? -static_cast<double>(rope->factor) : rope->factor};
}

void check_tokens(uint64_t tokens, uint64_t ld) {
    BSQ_REQUIRE(tokens <= 0x7FFFFFFFull, "kv4: too many tokens");
    BSQ_REQUIRE(ld <= 1ull << 28, "kv4: rows too far apart");
}

}  // namespace
}  // namespace bsq

using namespace bsq;

extern "C" {

uint64_t bsq_kv4_cache_bytes(uint64_t pages, uint32_t page, uint32_t heads, uint32_t dim) {
    return size_query([&] {
        const bsq_kv4_cache_t c{nullptr, pages, page, heads, dim};
        const Kv4Cache k = kv4_cache(&c, false);
        return pages * heads * static_cast<uint64_t>(k.head_bytes);
    });
}

uint64_t bsq_kv4_plan_workspace(uint32_t requests) {
    return size_query([&] {
        BSQ_REQUIRE(requests <= kPlanMostRequests, "kv4 plan: up to 16384 requests");
        return round256((static_cast<uint64_t>(requests) + 1) * 4);
    });
}

int bsq_kv4_plan(const int32_t *d_lengths, const int32_t *d_new, uint32_t requests, int32_t *d_table, uint32_t width,
                 uint32_t page, int32_t *d_free, uint64_t pages, const int32_t *d_free_count, int32_t *d_lengths_out,
                 int32_t *d_left, int32_t *d_starts, uint64_t tokens, int32_t *d_requests, int32_t *d_positions,
                 int32_t *d_slots, void *d_work, uint64_t work_bytes, void *stream) {
    return entry([&] {
        BSQ_REQUIRE(requests <= kPlanMostRequests, "kv4 plan: up to 16384 requests");
        const bsq_kv4_cache_t c{nullptr, pages, page, 1, 1};
        const Kv4Cache k = kv4_cache(&c, false);
        BSQ_REQUIRE(static_cast<uint64_t>(requests) * width <= 0x7FFFFFFFull, "kv4 plan: the table is too large");
        BSQ_REQUIRE(static_cast<uint64_t>(width) << k.shift <= 0x7FFFFFFFull, "kv4 plan: rows of the table are too long");
        BSQ_REQUIRE(tokens <= 0x7FFFFFFFull, "kv4 plan: too many tokens");
        BSQ_REQUIRE(d_free_count != nullptr && d_left != nullptr && d_starts != nullptr, "kv4 plan: null argument");
        BSQ_REQUIRE(requests == 0 || (d_lengths != nullptr && d_new != nullptr && d_lengths_out != nullptr), "kv4 plan: null argument");
        BSQ_REQUIRE(requests == 0 || width == 0 || d_table != nullptr, "kv4 plan: null table");
        BSQ_REQUIRE(pages == 0 || d_free != nullptr, "kv4 plan: null stack");
        BSQ_REQUIRE(tokens == 0 || (d_positions != nullptr && d_slots != nullptr), "kv4 plan: null output");
        check_work(d_work, work_bytes, round256((static_cast<uint64_t>(requests) + 1) * 4));
        const PlanArgs a{d_lengths,     d_new,  requests, d_table,  width, k.shift, d_free, static_cast<uint32_t>(pages),
                         d_free_count,  d_lengths_out, d_left, d_starts, static_cast<uint32_t>(tokens), d_requests,
                         d_positions, d_slots, static_cast<int32_t *>(d_work)};
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (requests <= kPlanThreads && tokens <= kPlanOneLaunch) {
            kv4_plan_kernel<true><<<1, kPlanThreads, 0, s>>>(a);
        } else {
            kv4_plan_kernel<false><<<1, kPlanThreads, 0, s>>>(a);
            BSQ_HIP(hipGetLastError());
            if (tokens > 0)
                kv4_places_kernel<<<static_cast<unsigned>(std::min<uint64_t>(ceil_div(tokens, kPlaceThreads), 4096)),
                                    kPlaceThreads, (requests + 1) * 4, s>>>(a);
        }
        BSQ_HIP(hipGetLastError());
    });
}

int bsq_rope_frequencies(uint32_t dims, double base, int scaling, double stretch, double length, double *frequencies,
                         float *factor) {
    return entry([&] {
        BSQ_REQUIRE(dims >= 2 && dims % 2 == 0 && dims <= kKv4MaxDim, "rope: an even number of dims, 2 to 256");
        BSQ_REQUIRE(base > 1.0 && std::isfinite(base), "rope: a base above 1");
        BSQ_REQUIRE(scaling >= 0 && scaling <= 3, "rope: unknown scaling");
        BSQ_REQUIRE(scaling == 0 || (stretch >= 1.0 && std::isfinite(stretch)), "rope: a stretch of 1 or more");
        BSQ_REQUIRE(scaling != 2 || dims > 2, "rope: this scaling takes 4 dims or more");
        BSQ_REQUIRE(scaling != 3 || (length > 0.0 && std::isfinite(length)), "rope: a length above zero");
        BSQ_REQUIRE(frequencies != nullptr && factor != nullptr, "rope: null output");
        constexpr double pi = 3.14159265358979323846;
        const double d = dims;
        const double b = scaling == 2 ? base * std::pow(stretch, d / (d - 2.0)) : base;
        // the pair that turns `turns` times in `length` positions
        const auto pair = [&](double turns) { return d * std::log(length / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
        const double low = std::max(0.0, std::floor(scaling == 3 ? pair(32.0) : 0.0));
        const double high = std::min(d - 1.0, std::ceil(scaling == 3 ? pair(1.0) : 0.0));
        for (uint32_t i = 0; i < dims / 2; ++i) {
            double f = std::pow(b, -2.0 * i / d);
            if (scaling == 1) f /= stretch;
            if (scaling == 3) {
                const double keep = 1.0 - std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
                f *= keep + (1.0 - keep) / stretch;
            }
            frequencies[i] = f;
        }
        *factor = scaling == 3 ? static_cast<float>(1.0 + 0.1 * std::log(stretch)) : 1.0f;
    });
}

int bsq_rope(const bsq_rope_t *rope, const int32_t *d_positions, const void *d_x, int type, uint64_t tokens, uint32_t heads,
             uint32_t dim, uint64_t ldx, int back, void *d_out, uint64_t ldo, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        BSQ_REQUIRE(rope != nullptr, "rope: null rope");
        BSQ_REQUIRE(dim >= 1 && dim <= kKv4MaxDim, "rope: heads of 1 to 256 values");
        BSQ_REQUIRE(heads <= 65535, "rope: up to 65535 heads");
        const uint64_t width = static_cast<uint64_t>(heads) * dim;
        check_tokens(tokens, std::max(ldx, ldo));
        BSQ_REQUIRE(ldx >= width && ldo >= width, "rope: rows overlap");
        RowsArgs a{};
        a.turn = turn_of(rope, dim, back);
        if (tokens == 0 || heads == 0) return;
        BSQ_REQUIRE(d_positions != nullptr, "rope: null positions");
        check_dense(d_x, t, "rope: null input");
        check_dense(d_out, t, "rope: null output");
        a.in_place = d_x == d_out && ldx == ldo;
        BSQ_REQUIRE(a.in_place || !overlap(tokens, CallRows(d_x, ldx, width, t), CallRows(d_out, ldo, width, t)),
                    "rope: out overlaps x");
        a.positions = d_positions;
        a.tokens = tokens;
        a.dim = dim;
        a.q = static_cast<const uint8_t *>(d_x);
        a.qo = static_cast<uint8_t *>(d_out);
        a.ldq = ldx;
        a.ldqo = ldo;
        a.q_heads = heads;
        launch_rows(a, t, false, static_cast<hipStream_t>(stream));
    });
}

int bsq_kv4_append(const bsq_kv4_cache_t *cache, const bsq_rope_t *rope, const int32_t *d_positions, const int32_t *d_slots,
                   uint64_t tokens, int type, const void *d_q, uint32_t q_heads, uint64_t ldq, void *d_q_out, uint64_t ldqo,
                   const void *d_k, uint64_t ldk, const void *d_v, uint64_t ldv, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        RowsArgs a{};
        a.cache = kv4_cache(cache, tokens > 0);
        const uint64_t width = static_cast<uint64_t>(a.cache.heads) * a.cache.dim, q_width = static_cast<uint64_t>(q_heads) * a.cache.dim;
        BSQ_REQUIRE(q_heads <= 65535, "kv4 append: up to 65535 heads");
        check_tokens(tokens, std::max(std::max(ldq, ldqo), std::max(ldk, ldv)));
        BSQ_REQUIRE(ldk >= width && ldv >= width, "kv4 append: rows overlap");
        BSQ_REQUIRE(d_q == nullptr || (ldq >= q_width && ldqo >= q_width), "kv4 append: rows overlap");
        if (rope != nullptr) a.turn = turn_of(rope, a.cache.dim, 0);
        if (tokens == 0) return;
        BSQ_REQUIRE(rope == nullptr || d_positions != nullptr, "kv4 append: null positions");
        BSQ_REQUIRE(d_slots != nullptr, "kv4 append: null slots");
        check_dense(d_k, t, "kv4 append: null keys");
        check_dense(d_v, t, "kv4 append: null values");
        if (d_q != nullptr && q_heads > 0) {
            check_dense(d_q, t, "");
            check_dense(d_q_out, t, "kv4 append: null output");
            a.in_place = d_q == d_q_out && ldq == ldqo;
            BSQ_REQUIRE(a.in_place || !overlap(tokens, CallRows(d_q, ldq, q_width, t), CallRows(d_q_out, ldqo, q_width, t)),
                        "kv4 append: queries' output overlaps them");
            if (!(a.in_place && rope == nullptr)) {  // else nothing changes
                // other workgroups read those at the same time
                const CallRows out(d_q_out, ldqo, q_width, t);
                BSQ_REQUIRE(!overlap(tokens, out, CallRows(d_k, ldk, width, t)) && !overlap(tokens, out, CallRows(d_v, ldv, width, t)),
                            "kv4 append: queries' output overlaps keys or values");
                a.q = static_cast<const uint8_t *>(d_q);
                a.qo = static_cast<uint8_t *>(d_q_out);
                a.q_heads = q_heads;
            }
        }
        a.positions = d_positions;
        a.slots = d_slots;
        a.tokens = tokens;
        a.dim = a.cache.dim;
        a.ldq = ldq;
        a.ldqo = ldqo;
        a.k = static_cast<const uint8_t *>(d_k);
        a.ldk = ldk;
        a.v = static_cast<const uint8_t *>(d_v);
        a.ldv = ldv;
        launch_rows(a, t, true, static_cast<hipStream_t>(stream));
    });
}

int bsq_kv4_read(const bsq_kv4_cache_t *cache, const int32_t *d_slots, uint64_t tokens, int type, void *d_k, uint64_t ldk,
                 void *d_v, uint64_t ldv, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        const Kv4Cache c = kv4_cache(cache, tokens > 0);
        const uint64_t width = static_cast<uint64_t>(c.heads) * c.dim;
        check_tokens(tokens, std::max(ldk, ldv));
        BSQ_REQUIRE((d_k == nullptr || ldk >= width) && (d_v == nullptr || ldv >= width), "kv4 read: rows overlap");
        if (tokens == 0 || (d_k == nullptr && d_v == nullptr)) return;
        BSQ_REQUIRE(d_slots != nullptr, "kv4 read: null slots");
        if (d_k != nullptr) check_dense(d_k, t, "");
        if (d_v != nullptr) check_dense(d_v, t, "");
        BSQ_REQUIRE(d_k == nullptr || d_v == nullptr || !overlap(tokens, CallRows(d_k, ldk, width, t), CallRows(d_v, ldv, width, t)),
                    "kv4 read: keys and values overlap");
        const uint32_t eights = (c.dim + 7) / 8;
        uint32_t per = std::max(1u, 1024u / (c.heads * eights));
        while (per > 1 && tokens / per < 2ull * cu_count()) per /= 2;
        const uint64_t groups = ceil_div(tokens, per);
        BSQ_REQUIRE(groups <= 0xFFFFFFFFull / 512, "kv4: too many tokens");
        by_type(t, [&](auto ty) {
            const dim3 grid(static_cast<unsigned>(groups), d_k && d_v ? 2 : 1);
            kv4_read_kernel<decltype(ty)::value><<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(
                c, d_slots, tokens, per, Divisor(c.heads), Divisor(eights), static_cast<uint8_t *>(d_k), ldk,
                static_cast<uint8_t *>(d_v), ldv);
        });
        BSQ_HIP(hipGetLastError());
    });
}

}  // extern "C"
