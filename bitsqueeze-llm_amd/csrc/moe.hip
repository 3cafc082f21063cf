// Routing to experts and the experts' layer on MX4 weights: the choice of
// experts with its gradient, the pairs (token, expert) in the experts' order,
// the join of a token's experts, and the layer's forward and backward calls.
// Compiled with -ffp-contract=off: the choice hangs on the last bit of a score
// plus a bias, which is rounded as two operations.
#include "mx4.hpp"

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include <bitsqz_llm_c.h>

namespace bsq {
namespace {

constexpr uint32_t kMaxExperts = 1024, kMaxChosen = 64, kMaxGroups = 64;

// ---------------------------------------------------------------------------
// one wave's reductions through DPP moves; the result in every lane
// ---------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or(int other, int v) {
    return __builtin_amdgcn_update_dpp(other, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_or(float other, float v) {
    return __int_as_float(dpp_or<CTRL, ROWS>(__float_as_int(other), __float_as_int(v)));
}
__device__ __forceinline__ float from_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
// (the least integer, which max takes for nothing, for lanes that read none: the
// move then folds into the max)
constexpr int kLeast = static_cast<int>(0x80000000u);
__device__ __forceinline__ int wave_max(int v) {
    v = max(v, dpp_or<0xB1, 0xF>(kLeast, v));
    v = max(v, dpp_or<0x4E, 0xF>(kLeast, v));
    v = max(v, dpp_or<0x141, 0xF>(kLeast, v));
    v = max(v, dpp_or<0x140, 0xF>(kLeast, v));
    v = max(v, dpp_or<0x142, 0xA>(kLeast, v));
    v = max(v, dpp_or<0x143, 0xC>(kLeast, v));
    return __builtin_amdgcn_readlane(v, 63);
}
// over each aligned run of `lanes` (a power of two), in every lane of it
__device__ __forceinline__ int run_max(int v, uint32_t lanes) {
    if (lanes > 1) v = max(v, dpp_or<0xB1, 0xF>(kLeast, v));
    if (lanes > 2) v = max(v, dpp_or<0x4E, 0xF>(kLeast, v));
    if (lanes > 4) v = max(v, dpp_or<0x141, 0xF>(kLeast, v));
    if (lanes > 8) v = max(v, dpp_or<0x140, 0xF>(kLeast, v));
    if (lanes > 16) v = max(v, __shfl_xor(v, 16));
    if (lanes > 32) v = max(v, __shfl_xor(v, 32));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_or<0xB1, 0xF>(0.0f, v);
    v += dpp_or<0x4E, 0xF>(0.0f, v);
    v += dpp_or<0x141, 0xF>(0.0f, v);
    v += dpp_or<0x140, 0xF>(0.0f, v);
    v += dpp_or<0x142, 0xA>(-0.0f, v);
    v += dpp_or<0x143, 0xC>(-0.0f, v);
    return from_lane(v, 63);
}

// Keys as integers that order as the floats do (-0 as 0), and back.
constexpr int kShut = static_cast<int>(0x807FFFFFu);  // -infinity
__device__ __forceinline__ int key_of(float f) {
    const int b = __float_as_int(f + 0.0f);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float value_of(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7FFFFFFF)); }

template <Mx4Type T>
constexpr float kLowest = T == Mx4Type::F32 ? -FLT_MAX : T == Mx4Type::BF16 ? -0x1.FEp127f : -65504.0f;

struct RouteArgs {
    const void *logits;
    const float *bias;
    uint64_t tokens, ld;
    uint32_t experts, k, groups, kept;
    int sigmoid, renorm;
    float scale;
};

// A token's logits: expert e = lane * NV + i.  Experts that are closed to the
// token (at or below the type's lowest value, or NaN) and those past the end
// read -infinity.
template <Mx4Type T>
__device__ __forceinline__ float open_logit(float v) {
    return v > kLowest<T> ? fminf(v, FLT_MAX) : -INFINITY;
}
template <Mx4Type T, int NV>
__device__ __forceinline__ void load_logits(const RouteArgs &a, uint64_t t, uint32_t lane, float x[NV]) {
    const uint32_t e0 = lane * NV;
    const uint64_t at = t * a.ld + e0;
    if (e0 + NV <= a.experts) {
        if constexpr (T == Mx4Type::F32) {
            __builtin_memcpy(x, static_cast<const float *>(a.logits) + at, 4 * NV);
        } else {
            uint16_t h[NV];
            __builtin_memcpy(h, static_cast<const uint16_t *>(a.logits) + at, 2 * NV);
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i] = T == Mx4Type::BF16 ? bf16_value(h[i]) : f16_value(h[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = open_logit<T>(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            x[i] = e0 + i < a.experts ? open_logit<T>(load_value<T>(a.logits, at + i)) : -INFINITY;
    }
}

__device__ __forceinline__ float sigmoid_of(float x) { return 1.0f / (1.0f + expf(-x)); }

// Softmax over the open experts: the largest logit and the sum of the
// exponentials (1 where there is none).
template <int NV>
__device__ __forceinline__ void softmax_of(const float x[NV], float e[NV], float &top, float &sum) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, x[i]);
    top = value_of(wave_max(key_of(m)));
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        e[i] = x[i] > -INFINITY ? expf(x[i] - top) : 0.0f;
        s += e[i];
    }
    sum = fmaxf(wave_sum(s), 1.0f);
}

// A lane's keys in descending order, equal ones by their index: value q of the
// list and its index in the q-th four bits of `where`.  Only neighbours change
// places, so that equal keys keep their order.  Lists longer than four are not
// sorted: their largest is found again each time.
template <int NV>
struct Keys {
    int key[NV];
    uint32_t where = 0x3210u;
    static constexpr bool kSorted = NV <= 4;
    // from any order: again where keys of the list were closed
    __device__ __forceinline__ void sort() {
        if constexpr (kSorted) {
            uint32_t at[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) at[i] = (where >> (4 * i)) & 15u;
            where = 0;
#pragma unroll
            for (int r = 0; r < NV; ++r)
#pragma unroll
                for (int i = r & 1; i + 1 < NV; i += 2) {
                    const bool swap = key[i + 1] > key[i];
                    const int hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
                    const uint32_t a = at[i], b = at[i + 1];
                    at[i] = swap ? b : a;
                    at[i + 1] = swap ? a : b;
                    key[i] = hi;
                    key[i + 1] = lo;
                }
#pragma unroll
            for (int i = 0; i < NV; ++i) where |= at[i] << (4 * i);
        }
    }
    // the largest key and its index
    __device__ __forceinline__ int head(uint32_t &at) const {
        if constexpr (kSorted) {
            at = where & 15u;
            return key[0];
        }
        int m = key[0];
        at = 0;
#pragma unroll
        for (int i = 1; i < NV; ++i) {
            at = key[i] > m ? i : at;
            m = max(m, key[i]);
        }
        return m;
    }
    __device__ __forceinline__ void drop(bool mine, uint32_t at) {
        if constexpr (kSorted) {
#pragma unroll
            for (int i = 0; i + 1 < NV; ++i) key[i] = mine ? key[i + 1] : key[i];
            key[NV - 1] = mine ? kShut : key[NV - 1];
            where = mine ? where >> 4 : where;
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) key[i] = mine && at == static_cast<uint32_t>(i) ? kShut : key[i];
        }
    }
};

// Lane l's keys of groups that are not among the `kept` best become kShut.
// A group's score: its largest key, with a bias the sum of its two largest.
template <int NV>
__device__ __forceinline__ void keep_groups(const RouteArgs &a, uint32_t lane, Keys<NV> &keys) {
    const uint32_t each = a.experts / a.groups, run = each / NV;
    const bool two = a.bias != nullptr;
    if (Keys<NV>::kSorted && each % NV == 0 && (run & (run - 1)) == 0) {
        // a group is an aligned run of lanes: all groups at once
        const int best = run_max(keys.key[0], run);
        int score = best;
        if (two) {
            const bool top = keys.key[0] == best;
            const int other = top ? (NV > 1 ? keys.key[NV > 1 ? 1 : 0] : kShut) : keys.key[0];
            int next = run_max(other, run);
            const uint64_t tied = (__ballot(top) >> (lane & ~(run - 1))) & (run == 64 ? ~0ull : (1ull << run) - 1);
            next = __builtin_popcountll(tied) > 1 ? best : next;
            score = next > kShut ? key_of(value_of(best) + value_of(next)) : best;
        }
        // its rank: groups above it, and equal ones of a lower number
        const uint32_t mine = lane / run;
        uint32_t rank = 0;
        for (uint32_t g = 0; g < a.groups; ++g) {
            const int s = __builtin_amdgcn_readlane(score, static_cast<int>(g * run));
            rank += s > score - (g < mine ? 1 : 0);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) keys.key[i] = rank < a.kept ? keys.key[i] : kShut;
        return;
    }
    uint32_t group[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) group[i] = (lane * NV + (Keys<NV>::kSorted ? (keys.where >> (4 * i)) & 15u : i)) / each;
    int of_group = kShut;
    for (uint32_t g = 0; g < a.groups; ++g) {
        int m = kShut;
        uint32_t at = NV;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool more = group[i] == g && keys.key[i] > m;
            m = more ? keys.key[i] : m;
            at = more ? i : at;
        }
        const int best = wave_max(m);
        int s = best;
        if (two && best > kShut) {
            const bool first = lane == static_cast<uint32_t>(__builtin_ctzll(__ballot(m == best)));
            m = kShut;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (group[i] == g && !(first && at == static_cast<uint32_t>(i))) m = max(m, keys.key[i]);
            const int next = wave_max(m);
            s = next > kShut ? key_of(value_of(best) + value_of(next)) : best;
        }
        of_group = lane == g ? s : of_group;
    }
    uint64_t chosen = 0;
    bool taken = lane >= a.groups;
    for (uint32_t j = 0; j < a.kept; ++j) {
        const int best = wave_max(taken ? kShut : of_group);
        const uint64_t at = __ballot(!taken && of_group == best);
        if (at == 0) break;
        const int g = __builtin_ctzll(at);
        chosen |= 1ull << g;
        taken |= lane == static_cast<uint32_t>(g);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) keys.key[i] = group[i] < 64 && ((chosen >> group[i]) & 1) ? keys.key[i] : kShut;
    keys.sort();  // a lane's keys may be of two groups: the open ones to the front
}

// One wave a token, NV experts a lane.  The largest of the lanes' largest keys
// is a DPP reduction of integers; the lowest lane that holds it gives the
// expert, so that ties go to the lowest.  Lane j then forms the weight of the
// j-th choice from that expert's own logit.  Scores and sums are FP32.
// Instructions bound it: 16384 tokens, 256 experts BF16, 8 groups, 8 chosen by
// sigmoid and bias 17 us (9 MB), half of it the eight rounds of a maximum; one
// wave a token as its logits are then in registers, and no round waits for a
// barrier.
template <Mx4Type T, int NV>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a, int32_t *__restrict__ ids,
                                                        float *__restrict__ weights) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;  // whole waves
    float x[NV], score[NV], top = 0.0f, sum = 1.0f;
    load_logits<T, NV>(a, t, lane, x);
    Keys<NV> keys;
    if (!a.sigmoid) {
        softmax_of<NV>(x, score, top, sum);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        keys.key[i] = key_of(x[i]);
        if (a.bias != nullptr && x[i] > -INFINITY) {
            const float v = (a.sigmoid ? sigmoid_of(x[i]) : score[i] / sum) + a.bias[lane * NV + i];
            keys.key[i] = v > -INFINITY ? key_of(v) : kShut;
        }
    }
    keys.sort();
    if (a.groups > 1) keep_groups<NV>(a, lane, keys);
    int32_t id = -1;
    for (uint32_t j = 0; j < a.k; ++j) {
        uint32_t at;
        const int m = keys.head(at);
        const int best = wave_max(m);
        if (best == kShut) break;  // uniform: no expert is left
        const int from = __builtin_ctzll(__ballot(m == best));
        const int32_t e = from * NV + __builtin_amdgcn_readlane(static_cast<int>(at), from);
        id = lane == j ? e : id;
        keys.drop(lane == static_cast<uint32_t>(from), at);
    }
    float mine = 0.0f;
    if (id >= 0) {
        const float v = open_logit<T>(load_value<T>(a.logits, t * a.ld + id));
        mine = a.sigmoid ? sigmoid_of(v) : expf(v - top) / sum;
    }
    const float total = a.renorm ? fmaxf(wave_sum(mine), FLT_MIN) : 1.0f;
    if (lane < a.k) {
        ids[t * a.k + lane] = id;
        weights[t * a.k + lane] = mine / total * a.scale;
    }
}

// d logits from d weights.  Lane j forms the score of the token's j-th expert
// again from its own logit.  With g = scale dw and w_j = s_j / S (S = 1 without
// the renormalisation) the gradient of the j-th expert's own logit is w_j h_j,
// h_j = g_j - sum g w, for sigmoid times 1 - s_j; for softmax every expert of
// score s loses s sum w h, which is 0 where the weights are renormalised.  Where
// S is held at the smallest normal number it does not depend on the scores, and
// h_j = g_j.  Nothing is divided by S but the scores, so no quotient overflows.
// The chosen reach their experts' lanes through a row in LDS.  The same tokens:
// 7.0 us (9.4 MB written; softmax reads as much), launch and latency.
template <Mx4Type T, int NV>
__global__ __launch_bounds__(256) void moe_route_backward_kernel(RouteArgs a, const int32_t *__restrict__ ids,
                                                                 const float *__restrict__ d_weights,
                                                                 void *__restrict__ d_logits, uint64_t ldd) {
    __shared__ float rows[4][64 * NV];
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;  // whole waves, which share nothing
    float *row = rows[threadIdx.x >> 6];
    float score[NV], top = 0.0f, sum = 1.0f;
    if (!a.sigmoid) {
        float x[NV];
        load_logits<T, NV>(a, t, lane, x);
        softmax_of<NV>(x, score, top, sum);
#pragma unroll
        for (int i = 0; i < NV; ++i) score[i] /= sum;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) row[lane * NV + i] = 0.0f;
    const int32_t id = lane < a.k ? ids[t * a.k + lane] : -1;
    float s = 0.0f, rest = 0.0f, d = 0.0f;
    bool real = static_cast<uint32_t>(id) < a.experts;
    if (real) {
        const float v = open_logit<T>(load_value<T>(a.logits, t * a.ld + id));
        real = v > -INFINITY;
        if (real) {
            s = a.sigmoid ? sigmoid_of(v) : expf(v - top) / sum;
            rest = a.sigmoid ? sigmoid_of(-v) : 0.0f;  // 1 - s, without the difference
            d = d_weights[t * a.k + lane] * a.scale;
        }
    }
    float share = s, mean = 0.0f;
    bool whole = false;  // the shares sum to one whatever the scores
    if (a.renorm) {
        const float total = wave_sum(s);
        whole = total > FLT_MIN;
        share = s / fmaxf(total, FLT_MIN);
        const float common = wave_sum(d * share);
        d = real && whole ? d - common : d;
    }
    if (!a.sigmoid && !whole) mean = wave_sum(d * share);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (real) row[id] = d * share * (a.sigmoid ? rest : 1.0f);  // a choice has an expert once
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        g[i] = row[lane * NV + i];
        if (!a.sigmoid) g[i] -= score[i] * mean;
    }
    const uint32_t e0 = lane * NV;
    const uint64_t at = t * ldd + e0;
    if (e0 + NV <= a.experts) {
        if constexpr (T == Mx4Type::F32) {
            __builtin_memcpy(static_cast<float *>(d_logits) + at, g, 4 * NV);
        } else {
            uint16_t h[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) h[i] = static_cast<uint16_t>(T == Mx4Type::BF16 ? bf16_bits(g[i]) : f16_bits(g[i]));
            __builtin_memcpy(static_cast<uint16_t *>(d_logits) + at, h, 2 * NV);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (e0 + i < a.experts) store_value<T>(d_logits, at + i, g[i]);
    }
}

// Pairs in the experts' order, the pairs of one expert by their number; those
// of no expert last.  Workgroup e counts the pairs of lower experts and its own
// (each wave a contiguous share), then writes its own in order: reads from
// cache only, no workspace and no atomics.  The ids of up to 16384 pairs (16 a
// lane) stay in registers; more are read again a tile at a time.  Latency bound
// (16384 pairs of 32 experts: 6 us, behind the encode of the tokens 0).
constexpr uint32_t kPlanThreads = 1024, kPlanEach = 16, kPlanTile = kPlanThreads * kPlanEach;

__device__ __forceinline__ void plan_expert(const int32_t *__restrict__ ids, uint32_t pairs, uint32_t experts, uint32_t e,
                                            int32_t *__restrict__ offsets, int32_t *__restrict__ order) {
    constexpr uint32_t kWaves = kPlanThreads / 64;
    __shared__ uint32_t lower[kWaves], own[2][kWaves];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t v[kPlanEach];
    auto load = [&](uint32_t base) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < kPlanEach; ++i) {
            const uint32_t p = base + wave * (64 * kPlanEach) + 64 * i + lane;
            const uint32_t id = p < pairs ? static_cast<uint32_t>(ids[p]) : 0u;
            v[i] = p < pairs ? min(id, experts) : 0xFFFFFFFFu;
        }
    };
    uint32_t lt = 0;
    for (uint32_t base = 0; base < pairs; base += kPlanTile) {
        load(base);
#pragma unroll
        for (uint32_t i = 0; i < kPlanEach; ++i) lt += __builtin_popcountll(__ballot(v[i] < e));
    }
    if (lane == 0) lower[wave] = lt;
    __syncthreads();
    uint32_t at = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) at += lower[w];
    if (threadIdx.x == 0) offsets[e] = static_cast<int32_t>(at);
    uint32_t turn = 0;
    for (uint32_t base = 0; base < pairs; base += kPlanTile, turn ^= 1) {
        if (pairs > kPlanTile) load(base);
        uint32_t eq = 0;
#pragma unroll
        for (uint32_t i = 0; i < kPlanEach; ++i) eq += __builtin_popcountll(__ballot(v[i] == e));
        if (lane == 0) own[turn][wave] = eq;
        __syncthreads();
        uint32_t to = at;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            to += w < wave ? own[turn][w] : 0u;
            at += own[turn][w];
        }
#pragma unroll
        for (uint32_t i = 0; i < kPlanEach; ++i) {
            const uint64_t who = __ballot(v[i] == e);
            if (v[i] == e)
                order[to + __builtin_popcountll(who & ((1ull << lane) - 1))] =
                    static_cast<int32_t>(base + wave * (64 * kPlanEach) + 64 * i + lane);
            to += __builtin_popcountll(who);
        }
    }
}

__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(const int32_t *__restrict__ ids, uint32_t pairs,
                                                                uint32_t experts, int32_t *__restrict__ offsets,
                                                                int32_t *__restrict__ order) {
    plan_expert(ids, pairs, experts, blockIdx.x, offsets, order);
}

// The plan by the first experts + 1 workgroups and the tokens' rows to MX4 by
// the others: neither needs the other, and a launch of its own costs more (4096
// x 4096 BF16 and 16384 pairs: 16.8 us).
template <Mx4Type T>
__global__ __launch_bounds__(kPlanThreads) void moe_begin_kernel(const int32_t *__restrict__ ids, uint32_t pairs,
                                                                 uint32_t experts, int32_t *__restrict__ offsets,
                                                                 int32_t *__restrict__ order, Mx4Rows rows) {
    if (blockIdx.x <= experts) plan_expert(ids, pairs, experts, blockIdx.x, offsets, order);
    else encode_rows<T, kPlanThreads>(rows, blockIdx.x - experts - 1, gridDim.x - experts - 1);
}

// out[t] = sum over the token's experts of weight * y, in the pairs' order; a
// lane takes eight columns.  HBM bound: 16384 rows of 2752 BF16 to 4096 19.8 us
// (113 MB; 21.8 at the rate of a large copy, part of y is still in cache).  y
// itself is of the type the caller asks for: in BF16 its rounding is as large
// as the output's own and independent of it, so the error grows by up to the
// square root of two, and half the bytes are moved; in FP16 a product above
// 65504 is infinite here whatever its weight.
template <Mx4Type Y, Mx4Type O>
__global__ __launch_bounds__(256) void moe_combine_kernel(const void *__restrict__ y, uint64_t tokens, uint32_t k,
                                                          uint32_t cols, uint32_t chunks,
                                                          const int32_t *__restrict__ ids,
                                                          const float *__restrict__ weights, uint32_t experts,
                                                          void *__restrict__ out, uint64_t ld) {
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t t = item / chunks;
    if (t >= tokens) return;
    const uint32_t c = 8 * static_cast<uint32_t>(item - t * chunks), valid = cols - c;
    float sum[8] = {};
#pragma unroll 4
    for (uint32_t j = 0; j < k; ++j) {
        // loads without a branch, so that several pairs' are in flight
        const uint64_t p = t * k + j;
        const bool real = static_cast<uint32_t>(ids[p]) < experts;
        const float w = weights[p];
        float v[8];
        load8<Y>(y, p * cols + c, valid, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = real ? __builtin_fmaf(w, v[i], sum[i]) : sum[i];
    }
    store8<O>(out, t * ld + c, valid, sum);
}

// d weights: a wave takes a pair's dot product with the token's d out.  4096
// pairs of 2752, y FP32 and d out BF16: 10.7 us for 56 MB (10.9 at the rate of a
// large copy; y comes in part from the last cache); loads of several pieces in
// flight take 10.4.
template <Mx4Type Y, Mx4Type D>
__global__ __launch_bounds__(256) void moe_weights_backward_kernel(const void *__restrict__ y, uint64_t pairs, uint32_t k,
                                                                   uint32_t cols, const int32_t *__restrict__ ids,
                                                                   uint32_t experts, const void *__restrict__ d_out,
                                                                   uint64_t ld, float *__restrict__ d_weights) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t p = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (p >= pairs) return;
    float sum = 0.0f;
    if (static_cast<uint32_t>(ids[p]) < experts) {
        const uint64_t t = p / k;
        for (uint32_t c = 8 * lane; c < cols; c += 512) {
            float a[8], b[8];
            load8<Y>(y, p * cols + c, cols - c, a);
            load8<D>(d_out, t * ld + c, cols - c, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(a[i], b[i], sum);
        }
    }
    sum = wave_sum(sum);
    if (lane == 0) d_weights[p] = sum;
}

template <class F>
void by_experts(uint32_t experts, F &&f) {
    if (experts <= 64) f(std::integral_constant<int, 1>{});
    else if (experts <= 128) f(std::integral_constant<int, 2>{});
    else if (experts <= 256) f(std::integral_constant<int, 4>{});
    else if (experts <= 512) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 16>{});
}

RouteArgs route_args(const void *logits, uint64_t tokens, uint32_t experts, uint64_t ld, const float *bias, int scoring,
                     Mx4Type type, uint32_t groups, uint32_t kept, uint32_t k, int renorm, float scale) {
    BSQ_REQUIRE(experts >= 1 && experts <= kMaxExperts, "moe route: 1 to 1024 experts");
    BSQ_REQUIRE(k >= 1 && k <= kMaxChosen && k <= experts, "moe route: 1 to 64 experts a token, at most all of them");
    BSQ_REQUIRE(scoring == 0 || scoring == 1, "moe route: scoring is 0 (softmax) or 1 (sigmoid)");
    BSQ_REQUIRE(groups >= 1 && groups <= kMaxGroups && experts % groups == 0, "moe route: groups (1 to 64) divide the experts");
    BSQ_REQUIRE(kept >= 1 && kept <= groups, "moe route: 1 to all groups are kept");
    BSQ_REQUIRE(ld >= experts, "moe route: rows overlap");
    BSQ_REQUIRE(tokens <= 0x7FFFFFFFull, "moe route: too many tokens");
    if (tokens > 0) check_dense(logits, type, "moe route: null logits");
    return {logits, bias, tokens, ld, experts, k, groups, kept, scoring, renorm != 0, scale};
}

void plan(const int32_t *ids, uint64_t pairs, uint32_t experts, int32_t *offsets, int32_t *order, hipStream_t stream) {
    moe_plan_kernel<<<experts + 1, kPlanThreads, 0, stream>>>(ids, static_cast<uint32_t>(pairs), experts, offsets, order);
    BSQ_HIP(hipGetLastError());
}

// A call's rows in as many launches as their threads' 32 bits ask for (one, but
// for tens of millions of rows; a loop in the kernels took 3 to 15 per cent more
// of their time): fn(first, count, groups) for `per` threads a row, workgroups of
// 256.
template <class F>
void in_turns(uint64_t rows, uint64_t per, F &&fn) {
    const uint64_t most = (1ull << 31) / per;
    for (uint64_t first = 0; first < rows; first += most) {
        const uint64_t count = std::min(most, rows - first);
        fn(first, count, static_cast<unsigned>(ceil_div(count * per, 256)));
    }
}
const uint8_t *row_of(const void *p, Mx4Type type, uint64_t row, uint64_t ld) {
    return static_cast<const uint8_t *>(p) + row * ld * type_bytes(type);
}
uint8_t *row_of(void *p, Mx4Type type, uint64_t row, uint64_t ld) {
    return static_cast<uint8_t *>(p) + row * ld * type_bytes(type);
}

void combine(const void *y, Mx4Type y_type, uint64_t tokens, uint32_t k, uint32_t cols, const int32_t *ids,
             const float *weights, uint32_t experts, void *out, Mx4Type type, uint64_t ld, hipStream_t stream) {
    if (tokens == 0 || cols == 0) return;
    const uint32_t chunks = static_cast<uint32_t>(ceil_div(cols, 8));
    in_turns(tokens, chunks, [&](uint64_t t, uint64_t count, unsigned groups) {
        by_type(y_type, [&](auto ty) {
            by_type(type, [&](auto to) {
                moe_combine_kernel<decltype(ty)::value, decltype(to)::value><<<groups, 256, 0, stream>>>(
                    row_of(y, y_type, t * k, cols), count, k, cols, chunks, ids + t * k, weights + t * k, experts,
                    row_of(out, type, t, ld), ld);
            });
        });
    });
    BSQ_HIP(hipGetLastError());
}

void weights_backward(const void *y, Mx4Type y_type, uint64_t tokens, uint32_t k, uint32_t cols, const int32_t *ids,
                      uint32_t experts, const void *d_out, Mx4Type type, uint64_t ld, float *d_weights,
                      hipStream_t stream) {
    in_turns(tokens, 64ull * k, [&](uint64_t t, uint64_t count, unsigned groups) {
        by_type(y_type, [&](auto ty) {
            by_type(type, [&](auto td) {
                moe_weights_backward_kernel<decltype(ty)::value, decltype(td)::value><<<groups, 256, 0, stream>>>(
                    row_of(y, y_type, t * k, cols), count * k, k, cols, ids + t * k, experts, row_of(d_out, type, t, ld), ld,
                    d_weights + t * k);
            });
        });
    });
    BSQ_HIP(hipGetLastError());
}

// Pieces of a workspace, in order.
struct Arena {
    uint8_t *at;
    uint64_t left;
    uint8_t *take(uint64_t bytes) {
        bytes = round256(bytes);
        BSQ_REQUIRE(bytes <= left, "moe: workspace too small");
        uint8_t *p = at;
        at += bytes;
        left -= bytes;
        return p;
    }
};

void check_layer(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs, uint32_t experts) {
    BSQ_REQUIRE(experts >= 1 && experts <= kMaxExperts, "moe linear: 1 to 1024 experts");
    BSQ_REQUIRE(k >= 1 && k <= kMaxChosen, "moe linear: 1 to 64 experts a token");
    BSQ_REQUIRE(tokens <= 0x7FFFFFFFull / k, "moe linear: too many tokens");
    BSQ_REQUIRE(n >= 1 && inputs >= 1 && n <= (1u << 22) && inputs <= (1u << 22), "moe linear: 1 to 2^22 inputs and outputs");
}
uint64_t slot_slices(uint64_t pairs, uint32_t experts) { return pairs / kMx4Slice + std::min<uint64_t>(pairs, experts); }
uint64_t linear_work(uint64_t tokens, uint64_t inputs) { return packed_bytes(tokens, mx4_slices(inputs)); }
uint64_t linear_backward_work(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs, uint32_t experts) {
    const uint64_t slots = slot_slices(tokens * k, experts);
    return packed_bytes(tokens, mx4_slices(n)) + round256(tokens * k * inputs * 4) + packed_bytes(n, slots) +
           packed_bytes(inputs, slots);
}

}  // namespace
}  // namespace bsq

using namespace bsq;

extern "C" {

int bsq_moe_route(const void *d_logits, int type, uint64_t tokens, uint32_t experts, uint64_t ld, const float *d_bias,
                  int scoring, uint32_t groups, uint32_t kept, uint32_t k, int renormalise, float scale, int32_t *d_ids,
                  float *d_weights, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        const RouteArgs a = route_args(d_logits, tokens, experts, ld, d_bias, scoring, t, groups, kept, k, renormalise, scale);
        if (tokens == 0) return;
        BSQ_REQUIRE(d_ids != nullptr && d_weights != nullptr, "moe route: null output");
        in_turns(tokens, 64, [&](uint64_t first, uint64_t count, unsigned groups) {
            RouteArgs some = a;
            some.logits = row_of(d_logits, t, first, ld);
            some.tokens = count;
            by_type(t, [&](auto ty) {
                by_experts(experts, [&](auto nv) {
                    moe_route_kernel<decltype(ty)::value, decltype(nv)::value>
                        <<<groups, 256, 0, static_cast<hipStream_t>(stream)>>>(some, d_ids + first * k, d_weights + first * k);
                });
            });
        });
        BSQ_HIP(hipGetLastError());
    });
}

int bsq_moe_route_backward(const void *d_logits, int type, uint64_t tokens, uint32_t experts, uint64_t ld, int scoring,
                           uint32_t k, int renormalise, float scale, const int32_t *d_ids, const float *d_d_weights,
                           void *d_d_logits, uint64_t ldd, void *stream) {
    return entry([&] {
        const Mx4Type t = type_of(type);
        const RouteArgs a = route_args(d_logits, tokens, experts, ld, nullptr, scoring, t, 1, 1, k, renormalise, scale);
        BSQ_REQUIRE(ldd >= experts, "moe route: rows overlap");
        if (tokens == 0) return;
        BSQ_REQUIRE(d_ids != nullptr && d_d_weights != nullptr, "moe route: null argument");
        check_dense(d_d_logits, t, "moe route: null gradient");
        in_turns(tokens, 64, [&](uint64_t first, uint64_t count, unsigned groups) {
            RouteArgs some = a;
            some.logits = row_of(d_logits, t, first, ld);
            some.tokens = count;
            by_type(t, [&](auto ty) {
                by_experts(experts, [&](auto nv) {
                    moe_route_backward_kernel<decltype(ty)::value, decltype(nv)::value>
                        <<<groups, 256, 0, static_cast<hipStream_t>(stream)>>>(
                            some, d_ids + first * k, d_d_weights + first * k, row_of(d_d_logits, t, first, ldd), ldd);
                });
            });
        });
        BSQ_HIP(hipGetLastError());
    });
}

int bsq_moe_plan(const int32_t *d_ids, uint64_t pairs, uint32_t experts, int32_t *d_offsets, int32_t *d_order,
                 void *stream) {
    return entry([&] {
        BSQ_REQUIRE(experts >= 1 && experts <= kMaxExperts, "moe plan: 1 to 1024 experts");
        BSQ_REQUIRE(pairs <= 0x7FFFFFFFull, "moe plan: too many pairs");
        BSQ_REQUIRE(d_offsets != nullptr && (pairs == 0 || (d_ids != nullptr && d_order != nullptr)), "moe plan: null argument");
        plan(d_ids, pairs, experts, d_offsets, d_order, static_cast<hipStream_t>(stream));
    });
}

int bsq_moe_combine(const void *d_y, int y_type, uint64_t tokens, uint32_t k, uint64_t n, const int32_t *d_ids,
                    const float *d_weights, uint32_t experts, void *d_out, int type, uint64_t ld, void *stream) {
    return entry([&] {
        const Mx4Type ty = type_of(y_type), t = type_of(type);
        check_layer(tokens, k, n, 1, experts);
        BSQ_REQUIRE(ld >= n, "moe combine: rows overlap");
        if (tokens == 0) return;
        BSQ_REQUIRE(d_ids != nullptr && d_weights != nullptr, "moe combine: null argument");
        check_dense(d_y, ty, "moe combine: null argument");
        check_dense(d_out, t, "moe combine: null output");
        combine(d_y, ty, tokens, k, static_cast<uint32_t>(n), d_ids, d_weights, experts, d_out, t, ld,
                static_cast<hipStream_t>(stream));
    });
}

uint64_t bsq_moe_linear_workspace(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs, uint32_t experts) {
    return size_query([&] {
        check_layer(tokens, k, n, inputs, experts);
        return linear_work(tokens, inputs);
    });
}

int bsq_moe_linear(const void *d_x, int x_type, uint64_t tokens, uint64_t inputs, uint64_t ldx, const int32_t *d_ids,
                   const float *d_weights, uint32_t k, const uint8_t *d_w_codes, const uint8_t *d_w_scales,
                   uint32_t experts, uint64_t n, int32_t *d_offsets, int32_t *d_order, void *d_y, int y_type, void *d_out,
                   int out_type, uint64_t ldo, void *d_work, uint64_t work_bytes, void *stream) {
    return entry([&] {
        const Mx4Type tx = type_of(x_type), ty = type_of(y_type), to = type_of(out_type);
        check_layer(tokens, k, n, inputs, experts);
        BSQ_REQUIRE(ldx >= inputs && ldo >= n, "moe linear: rows overlap");
        BSQ_REQUIRE(d_offsets != nullptr, "moe linear: null argument");
        hipStream_t s = static_cast<hipStream_t>(stream);
        const uint64_t pairs = tokens * k;
        if (pairs > 0) {
            BSQ_REQUIRE(d_ids != nullptr && d_weights != nullptr && d_order != nullptr, "moe linear: null argument");
            check_dense(d_x, tx, "moe linear: null input");
            check_dense(d_y, ty, "moe linear: null y");
            check_dense(d_out, to, "moe linear: null output");
            check_packed(d_w_codes, d_w_scales);
            check_work(d_work, work_bytes, linear_work(tokens, inputs));
        }
        if (pairs == 0) {
            plan(d_ids, pairs, experts, d_offsets, d_order, s);
            return;
        }
        const uint32_t slices = static_cast<uint32_t>(mx4_slices(inputs));
        Arena arena{static_cast<uint8_t *>(d_work), work_bytes};
        uint8_t *codes = arena.take(tokens * slices * 128), *scales = arena.take(tokens * slices * 8);
        const Mx4Rows rows{static_cast<const uint8_t *>(d_x), tokens, inputs, ldx, 0, tokens, slices * (kMx4Slice / 8),
                           codes, scales};
        const uint64_t groups = grid_over(ceil_div(tokens * rows.chunks, kPlanThreads));
        Mx4Product p;
        p.a = {codes, scales};
        p.b = {d_w_codes, d_w_scales};
        p.M = static_cast<uint32_t>(pairs);
        p.N = static_cast<uint32_t>(n);
        p.slices = slices;
        p.out = d_y;
        p.type = ty;
        p.ld = n;
        p.offsets = d_offsets;
        p.order = d_order;
        p.experts = experts;
        p.per_token = k;
        check_mx4_product(p);
        by_type(tx, [&](auto t) {
            moe_begin_kernel<decltype(t)::value><<<static_cast<unsigned>(experts + 1 + groups), kPlanThreads, 0, s>>>(
                d_ids, static_cast<uint32_t>(pairs), experts, d_offsets, d_order, rows);
        });
        BSQ_HIP(hipGetLastError());
        launch_mx4_product(p, nullptr, 0, s);
        combine(d_y, ty, tokens, k, static_cast<uint32_t>(n), d_ids, d_weights, experts, d_out, to, ldo, s);
    });
}

uint64_t bsq_moe_linear_backward_workspace(uint64_t tokens, uint32_t k, uint64_t n, uint64_t inputs, uint32_t experts) {
    return size_query([&] {
        check_layer(tokens, k, n, inputs, experts);
        return linear_backward_work(tokens, k, n, inputs, experts);
    });
}

int bsq_moe_linear_backward(const void *d_d_out, int d_type, uint64_t tokens, uint64_t n, uint64_t ldd, const void *d_x,
                            int x_type, uint64_t inputs, uint64_t ldx, const int32_t *d_ids, const float *d_weights,
                            uint32_t k, const int32_t *d_offsets, const int32_t *d_order, const void *d_y, int y_type,
                            const uint8_t *d_wt_codes, const uint8_t *d_wt_scales, uint32_t experts, void *d_dx,
                            uint64_t lddx, float *d_d_weights, void *d_dw, int g_type, void *d_work, uint64_t work_bytes,
                            void *stream) {
    return entry([&] {
        const Mx4Type td = type_of(d_type), tx = type_of(x_type), ty = type_of(y_type), tg = type_of(g_type);
        check_layer(tokens, k, n, inputs, experts);
        BSQ_REQUIRE(ldd >= n && (d_dw == nullptr || ldx >= inputs) && (d_dx == nullptr || lddx >= inputs),
                    "moe linear: rows overlap");
        const uint64_t pairs = tokens * k;
        BSQ_REQUIRE(d_offsets != nullptr, "moe linear: null argument");
        if (pairs > 0) {
            check_dense(d_d_out, td, "moe linear: null gradient");
            BSQ_REQUIRE(d_ids != nullptr && d_weights != nullptr && d_order != nullptr, "moe linear: null argument");
            BSQ_REQUIRE(d_dx == nullptr || (d_wt_codes != nullptr && d_wt_scales != nullptr), "moe linear: dx needs the weights' columns");
            BSQ_REQUIRE(d_d_weights == nullptr || d_y != nullptr, "moe linear: the weights' gradient needs y");
            BSQ_REQUIRE(d_dw == nullptr || d_x != nullptr, "moe linear: dw needs x");
            if (d_dx) check_packed(d_wt_codes, d_wt_scales);
            if (d_dx) check_dense(d_dx, tg, "");
            if (d_d_weights) check_dense(d_y, ty, "");
            if (d_dw) check_dense(d_x, tx, "");
            // its rows of slots are 128 bytes a slice, and a tile's 256 of them lie
            // within 32 bits
            BSQ_REQUIRE(d_dw == nullptr || slot_slices(pairs, experts) <= 1u << 17, "moe linear: too many pairs for dw");
            check_work(d_work, work_bytes, linear_backward_work(tokens, k, n, inputs, experts));
        }
        if (d_dw) check_dense(d_dw, tg, "");
        hipStream_t s = static_cast<hipStream_t>(stream);
        const uint64_t slots = slot_slices(pairs, experts);
        const uint32_t slices = static_cast<uint32_t>(mx4_slices(n));
        Arena arena{static_cast<uint8_t *>(d_work), work_bytes};
        uint8_t *codes = nullptr, *scales = nullptr, *z = nullptr, *gc = nullptr, *gs = nullptr, *xc = nullptr, *xs = nullptr;
        if (pairs > 0) {
            codes = arena.take(tokens * slices * 128), scales = arena.take(tokens * slices * 8);
            z = arena.take(pairs * inputs * 4);
            gc = arena.take(n * slots * 128), gs = arena.take(n * slots * 8);
            xc = arena.take(inputs * slots * 128), xs = arena.take(inputs * slots * 8);
        }
        Mx4Product dx, dw;
        // dx[t] = sum of weight * (q(d out[t]) W_e): the layer itself, with
        // the weights' columns for their rows.  The terms are FP32 until they
        // are summed, whatever the gradients' type: a pair's product may lie
        // above FP16's range where its weight brings it back, and in BF16
        // dx was off by 0.0024 in place of 0.0017 (2048 tokens to 2 of 16
        // experts, 2752 and 2048: product and join 42 and 7.7 us, of BF16 terms
        // 32 and 6.1).
        dx.a = {codes, scales};
        dx.b = {d_wt_codes, d_wt_scales};
        dx.M = static_cast<uint32_t>(pairs);
        dx.N = static_cast<uint32_t>(inputs);
        dx.slices = slices;
        dx.out = z;
        dx.type = Mx4Type::F32;
        dx.ld = inputs;
        dx.offsets = d_offsets;
        dx.order = d_order;
        dx.experts = experts;
        dx.per_token = k;
        // dw[e] = the sum over the expert's pairs of q(weight d out)^T q(x),
        // both rounded in blocks of 32 pairs
        dw.a = {gc, gs};
        dw.b = {xc, xs};
        dw.M = static_cast<uint32_t>(n);
        dw.N = static_cast<uint32_t>(inputs);
        dw.slices = static_cast<uint32_t>(slots);
        dw.out = d_dw;
        dw.type = tg;
        dw.ld = inputs;
        dw.offsets = d_offsets;
        dw.experts = experts;
        dw.shared_slots = true;
        const bool at_once = d_dx != nullptr && d_dw != nullptr && td == tx;
        if (d_dx != nullptr) check_mx4_product(dx);
        if (d_dw != nullptr) check_mx4_product(dw);
        if (at_once) {
            check_mx4_encode_backward(td, n, inputs, tokens, slots);
        } else if (d_dw != nullptr) {
            check_mx4_encode_slots(td, n, slots);
            check_mx4_encode_slots(tx, inputs, slots);
        }
        if (pairs > 0) {
            Mx4Slots of{d_offsets, d_order, d_weights, experts, k};
            if (at_once) {
                launch_mx4_encode_backward(d_d_out, n, ldd, d_x, inputs, ldx, td, tokens, of, slots, gc, gs, xc, xs, codes,
                                           scales, s);
            } else {
                if (d_dx != nullptr) launch_mx4_encode(d_d_out, td, 1, tokens, n, ldd, 0, codes, scales, nullptr, nullptr, s);
                if (d_dw != nullptr) {
                    launch_mx4_encode_slots(d_d_out, td, n, ldd, of, slots, gc, gs, s);
                    of.weights = nullptr;
                    launch_mx4_encode_slots(d_x, tx, inputs, ldx, of, slots, xc, xs, s);
                }
            }
        }
        if (pairs > 0 && d_dx != nullptr) {
            launch_mx4_product(dx, nullptr, 0, s);
            combine(z, Mx4Type::F32, tokens, k, static_cast<uint32_t>(inputs), d_ids, d_weights, experts, d_dx, tg, lddx, s);
        }
        if (pairs > 0 && d_d_weights != nullptr)
            weights_backward(d_y, ty, tokens, k, static_cast<uint32_t>(n), d_ids, experts, d_d_out, td, ldd, d_d_weights, s);
        if (d_dw != nullptr) launch_mx4_product(dw, nullptr, 0, s);
    });
}

}  // extern "C"
