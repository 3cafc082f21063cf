// Attention over the paged MX4 cache: prompts and chunks of them
// (kv4_attention.hpp).
//
// 128 rows of queries (tokens times the heads of a group) share the keys: a
// workgroup of four waves converts 64 keys and values at a time to BF16 in LDS, once
// for all rows, and every wave multiplies them with 32 rows.  The next 64 are
// converted into a second buffer while these are multiplied, 16 by each wave, from
// words that were loaded a step earlier, at a page that was looked up two steps
// earlier and is the wave's alone, so that addresses are scalar.
//
// Products are S^T = K Q^T and O^T = V^T P^T on 32 x 32 tiles, so a lane holds one
// row of queries: its reference, sum and weights never leave it but to its partner
// 32 lanes on.  Lane l = 32 h + i holds of S^T's 32 keys those at 8 b + 4 h + r; the
// values' rows of 16 lie in LDS in the order 0-3, 8-11, 4-7, 12-15, so that the
// eight weights that a lane has are the eight that the next product wants of it.
//
// Bound by the matrix instructions and the vector ones between them, which two waves
// a SIMD overlap only in part: a prompt of 8192, 32 heads on 8 of 128, takes 613 to
// 655 us, 840 to 897 TFLOP/s (1173 in a large BF16 product of the library); a wave's
// 64 keys are 32 matrix instructions and some 240 others, 32 of them exponentials.
// Waves of raised priority during the products: 695 us against 669.  Tiles of 16 rows
// (kv4_few.hpp) take 2790.
#include "kv4_attention.hpp"

namespace bsq {
namespace {

constexpr int kThreads = kPromptThreads;
constexpr uint32_t kKeys = 64;

__device__ __forceinline__ uint32_t tiles_of(const AttentionArgs &a, const Request &q) {
    const uint64_t rows = static_cast<uint64_t>(q.count) * a.group;
    return rows <= a.few ? 0u : static_cast<uint32_t>((rows + kPromptRows - 1) / kPromptRows);
}

// What a lane converts of 16 keys and values: of one token a block of keys, and of
// the eight tokens whose weights a lane holds together four channels of values.
struct Raw {
    uint32_t k[4], ks, nan;
    uint32_t v[8], vs[4];
};

template <int NB, int P>
__global__ __launch_bounds__(kThreads, NB <= 4 && P <= 2 ? 2 : 1) void kv4_prompt_kernel(AttentionArgs a, uint32_t tiles) {
    constexpr int kUnits = 16 * NB, kRounds = (kUnits + 63) / 64;  // a wave's
    constexpr uint32_t kRow = 16 * NB;                             // bytes of a token's codes
    constexpr uint32_t kKeyRow = 32 * NB + 8, kValueRow = kKeys + 8;  // elements; 16 bytes on: other banks
    __shared__ __attribute__((aligned(16))) uint16_t keys[2][kKeys][kKeyRow];
    __shared__ __attribute__((aligned(16))) uint16_t vals[2][32 * NB][kValueRow];
    __shared__ uint8_t nans[2][kKeys * NB];
    __shared__ uint32_t bads[2][4];
    __shared__ uint32_t sums[kThreads / 64];
    __shared__ uint32_t found[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t heads = a.cache.heads, h = blockIdx.x % heads, rest = blockIdx.x / heads;
    // the last tiles of a prompt see most keys: they begin first
    const uint32_t share = rest % a.each, tile = tiles - 1 - rest / a.each;
    Split *split = a.each > 1 && share == 0 ? a.splits + static_cast<uint64_t>(tile) * heads + h : nullptr;

    // whose tile this is
    uint32_t r = 0, in = tile;
    if (a.requests > 1) {
        const uint32_t per = (a.requests + kThreads - 1) / kThreads;
        const uint32_t r_begin = min(tid * per, a.requests), r_end = min(r_begin + per, a.requests);
        uint32_t mine = 0;
        for (uint32_t i = r_begin; i < r_end; ++i) mine += tiles_of(a, load_request(a, i));
        uint32_t before = wave_prefix(mine);
        if (lane == 63) sums[wave] = before;
        if (tid == 0) found[0] = 0xFFFFFFFFu;
        __syncthreads();
        before -= mine;
        for (uint32_t w = 0; w < wave; ++w) before += sums[w];
        if (tile >= before && tile < before + mine) {
            uint32_t base = before;
            for (uint32_t i = r_begin; i < r_end; ++i) {
                const uint32_t n = tiles_of(a, load_request(a, i));
                if (tile < base + n) {
                    found[0] = i;
                    found[1] = tile - base;
                    break;
                }
                base += n;
            }
        }
        __syncthreads();
        r = __builtin_amdgcn_readfirstlane(found[0]);
        in = __builtin_amdgcn_readfirstlane(found[1]);
    }
    Request rq{0, 0, 0};
    if (r < a.requests) rq = load_request(a, r);
    if (r >= a.requests || in >= tiles_of(a, rq)) {
        if (split != nullptr && tid == 0) split->parts = 0;
        return;
    }
    const uint32_t row0 = in * kPromptRows, count = min(kPromptRows, static_cast<uint32_t>(rq.count) * a.group - row0);

    // what the tile's queries see, and this lane's
    const int32_t qa = static_cast<int32_t>(row0 / a.group), qb = static_cast<int32_t>((row0 + count - 1) / a.group);
    const int32_t past = rq.past(), window = static_cast<int32_t>(min(a.window, 0x7FFFFFFFu));
    const auto lim_of = [&](int32_t query) { return a.causal ? past + query + 1 : rq.length; };
    const auto low_of = [&](int32_t query) { return window ? max(past + query + 1, 0) - window : 0; };
    const int32_t any_lim = lim_of(qb), any_low = low_of(qa), all_lim = lim_of(qa), all_low = low_of(qb);
    const uint32_t i = lane & 31, half = lane >> 5, row = wave * 32 + i, mine = row0 + min(row, count - 1);
    const int32_t lim = lim_of(static_cast<int32_t>(mine / a.group)), low = low_of(static_cast<int32_t>(mine / a.group));
    const bool mixed = a.causal && qa != qb;
    const int32_t begin = max(any_low, 0) & ~static_cast<int32_t>(kKeys - 1);
    const uint32_t steps = any_lim > begin ? static_cast<uint32_t>(any_lim - begin + kKeys - 1) / kKeys : 0u;
    const uint32_t s0 = static_cast<uint32_t>(static_cast<uint64_t>(steps) * share / a.each);
    const uint32_t s1 = static_cast<uint32_t>(static_cast<uint64_t>(steps) * (share + 1) / a.each);
    // tables may end within the last kKeys of 31 bits, so nothing is added to t; a tile
    // with keys has all_lim above -kPromptRows
    const auto edge = [&](int32_t t) { return t > all_lim - static_cast<int32_t>(kKeys) || t < all_low; };

    // queries: lane (h, i) has row i's channels 16 s + 8 h .. + 8
    const uint64_t token = static_cast<uint32_t>(rq.first) + mine / a.group;
    const uint32_t head = h * a.group + mine % a.group;
    u32x4 q[P][2 * NB];
    {
        const uint64_t at = token * a.ldq + static_cast<uint64_t>(head) * a.cache.dim;
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            const uint32_t c = 16 * s + 8 * half;
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (row < count && c < a.cache.dim)
                by_device_type(a.q_type, [&](auto t) { load8<decltype(t)::value>(a.q, at + c, a.cache.dim - c, x); });
            if (a.negate) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = -x[e];
            }
            u32x4 w[P];
            pieces<P, true>(x, w);
#pragma unroll
            for (int p = 0; p < P; ++p) q[p][s] = w[p];
        }
    }
    f32x16 o[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
    float top = -__builtin_inff(), base = 0.0f, sum = 0.0f;

    // this wave's sixteen of a step, lane by lane: unit u of `kUnits`
    struct Unit {
        uint32_t token, block;    // of keys
        uint32_t half, quarter;   // of the tokens, of the channels (four) of values
        bool real;
    };
    const auto unit_of = [&](int n) {
        const uint32_t u = lane + 64 * n;
        return Unit{u / NB, u % NB, u & 1, u >> 1, kUnits % 64 == 0 || u < static_cast<uint32_t>(kUnits)};
    };
    // above zero, so that what is not seen stays at minus infinity; with the smallest
    // value scores of any size count as zero, to 2^-21
    const float factor = fmaxf(a.factor, 0x1p-149f);
    const uint32_t page_bytes = a.cache.head_bytes * heads;
    const uint8_t *const head0 = a.cache.pages + h * a.cache.head_bytes;
    const auto id_of = [&](int32_t t) { return page_of(a, r, rq, static_cast<uint32_t>(t) + 16 * wave); };
    const auto load_raw = [&](Raw raw[kRounds], uint32_t id, int32_t t) {
        const uint32_t in = (static_cast<uint32_t>(t) + 16 * wave) & (a.cache.page() - 1);
        const uint8_t *p = head0 + static_cast<uint64_t>(id >= a.cache.count ? 0u : id) * page_bytes;
        const uint8_t *keys_at = p + in * kRow, *values_at = keys_at + (kRow << a.cache.shift);
        const uint8_t *ks_at = p + (2 * kRow << a.cache.shift) + in * NB, *vs_at = ks_at + (NB << a.cache.shift);
#pragma unroll
        for (int n = 0; n < kRounds; ++n) {
            const Unit u = unit_of(n);
            if (!u.real) continue;
            Raw &w = raw[n];
            __builtin_memcpy(w.k, __builtin_assume_aligned(keys_at + (u.token * kRow + 16 * u.block), 16), 16);
            // words of four tokens' scales, the byte picked as it is used
            const uint32_t scale_at = 4 * ((u.token & 3) * NB + u.block);
            w.ks = *reinterpret_cast<const uint32_t *>(ks_at + scale_at);
            w.nan = mixed && edge(t) ? *reinterpret_cast<const uint32_t *>(vs_at + scale_at) : 0u;
            const uint32_t codes_at = 4 * u.half * kRow + 2 * u.quarter;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w.v[j] = *reinterpret_cast<const uint16_t *>(values_at + codes_at + ((j & 3) + 8 * (j >> 2)) * kRow);
#pragma unroll
            for (int j = 0; j < 4; ++j) w.vs[j] = *reinterpret_cast<const uint32_t *>(vs_at + 4 * (u.quarter >> 3) + j * 4 * NB);
        }
    };
    const auto convert = [&](Raw raw[kRounds], uint32_t id, int32_t t, uint32_t buffer) {
        const bool bad = id >= a.cache.count;
        if (lane == 0) bads[buffer][wave] = bad;
#pragma unroll
        for (int n = 0; n < kRounds; ++n) {
            const Unit u = unit_of(n);
            if (!u.real) continue;
            Raw &w = raw[n];
            const uint32_t token = 16 * wave + u.token;
            const uint32_t ks_shift = 8 * ((u.token >> 2) & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j) w.vs[j] >>= 8 * u.half;  // the token's byte lowest, that of the one eight on third
            if (edge(t) || bad) {
                if (mixed) nans[buffer][token * NB + u.block] = (w.nan >> ks_shift & 0xFFu) == 255u;
                // what no query sees may hold anything, NaN among it; a NaN block that
                // some see and others do not goes past the products
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int32_t at = t + static_cast<int32_t>(16 * wave + 4 * u.half + (j & 3) + 8 * (j >> 2));
                    const uint32_t shift = 16 * (j >> 2), byte = w.vs[j & 3] >> shift & 0xFFu;
                    if (at >= any_lim || at < any_low || bad || (mixed && byte == 255u)) {
                        w.v[j] = 0;
                        w.vs[j & 3] = (w.vs[j & 3] & ~(0xFFu << shift)) | 127u << shift;
                    }
                }
            }
            const float ks = __uint_as_float((w.ks >> ks_shift & 0xFFu) << 23);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const u32x4 x = {cvt(w.k[c], ks, 0), cvt(w.k[c], ks, 1), cvt(w.k[c], ks, 2), cvt(w.k[c], ks, 3)};
                *reinterpret_cast<u32x4 *>(&keys[buffer][token][32 * u.block + 8 * c]) = x;
            }
            float scale[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] = __uint_as_float((w.vs[j & 3] >> (16 * (j >> 2)) & 0xFFu) << 23);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                u32x4 even, odd;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t x0 = cvt(w.v[j], scale[j], c), x1 = cvt(w.v[j + 1], scale[j + 1], c);
                    even[j >> 1] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
                    odd[j >> 1] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
                }
                *reinterpret_cast<u32x4 *>(&vals[buffer][4 * u.quarter + 2 * c][16 * wave + 8 * u.half]) = even;
                *reinterpret_cast<u32x4 *>(&vals[buffer][4 * u.quarter + 2 * c + 1][16 * wave + 8 * u.half]) = odd;
            }
        }
    };

    if (s0 < s1) {
        const auto at = [&](uint32_t s) { return begin + static_cast<int32_t>(min(s, s1 - 1) * kKeys); };
        Raw raw[kRounds];
        uint32_t id = id_of(at(s0)), then = id_of(at(s0 + 1));  // of `raw`, and of the step behind it
        load_raw(raw, id, at(s0));
        convert(raw, id, at(s0), 0);
        id = then;
        load_raw(raw, id, at(s0 + 1));
        then = id_of(at(s0 + 2));
        __syncthreads();
        for (uint32_t s = s0; s < s1; ++s) {
            const uint32_t buffer = (s - s0) & 1;
            const int32_t t = at(s);
            f32x16 x[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[n][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const u32x4 k = *reinterpret_cast<const u32x4 *>(&keys[buffer][32 * n + i][16 * c + 8 * half]);
#pragma unroll
                    for (int p = 0; p < P; ++p) x[n] = mfma(k, q[p][c], x[n]);
                }
            if (s + 1 < s1) {
                convert(raw, id, at(s + 1), buffer ^ 1);
                id = then;
                load_raw(raw, id, at(s + 2));
                then = id_of(at(s + 3));
            }
            const uint32_t bad = bads[buffer][0] | bads[buffer][1] << 1 | bads[buffer][2] << 2 | bads[buffer][3] << 3;
            const bool masked = edge(t) || __builtin_amdgcn_readfirstlane(bad) != 0;
            if (masked) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int32_t key = t + static_cast<int32_t>(32 * n + 8 * (e >> 2) + 4 * half + (e & 3));
                        if (key >= lim || key < low || (bad >> (2 * n + (e >> 3)) & 1)) x[n][e] = -__builtin_inff();
                    }
                if (mixed && edge(t)) {
                    uint32_t any = 0;
                    for (uint32_t u = lane; u < kKeys * NB; u += 64) any |= nans[buffer][u];
                    if (__any(any != 0))
                        for (uint32_t key = 0; key < kKeys; ++key) {
                            const int32_t where = t + static_cast<int32_t>(key);
                            if (where >= lim || where < low || (bad >> (key >> 4) & 1)) continue;
#pragma unroll
                            for (int c = 0; c < NB; ++c)
                                if (nans[buffer][key * NB + c]) {
#pragma unroll
                                    for (int e = 0; e < 16; ++e) o[c][e] = __builtin_nanf("");
                                }
                        }
                }
            }
            float high = x[0][0];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) high = fmaxf(high, x[n][e]);
            high *= factor;
            if (__any(high > top + kSlack)) {
                high = fmaxf(high, __shfl_xor(high, 32));
                const float now = fmaxf(top, high), keep = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
                sum *= keep;
#pragma unroll
                for (int c = 0; c < NB; ++c) o[c] *= keep;
                top = now;
                base = now == -__builtin_inff() ? 0.0f : now;
            }
            u32x4 pw[4][P];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float score = x[m >> 1][8 * (m & 1) + e];
                    w[e] = __builtin_amdgcn_exp2f(fmaf(score, factor, -base));
                    sum += w[e];
                }
                pieces<P>(w, pw[m]);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(&vals[buffer][32 * c + i][16 * m + 8 * half]);
#pragma unroll
                    for (int p = 0; p < P; ++p) o[c] = mfma(v, pw[m][p], o[c]);
                }
            __syncthreads();
        }
    }

    sum += __shfl_xor(sum, 32);
    if (split != nullptr && tid == 0) {
        const uint32_t first = (tile * heads + h) * a.each;
        *split = {a.each, first, first + 1, 1, h, row0, count, static_cast<uint32_t>(rq.first)};
    }
    if (row >= count) return;
    if (a.each > 1) {
        float *p = a.parts + ((static_cast<uint64_t>(tile) * heads + h) * a.each + share) * (kPromptRows * part_row(NB)) + row * part_row(NB);
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x4 v = {o[c][e], o[c][e + 1], o[c][e + 2], o[c][e + 3]};
                *reinterpret_cast<f32x4 *>(p + 32 * c + 2 * e + 4 * half) = v;
            }
        if (half == 0) {
            p[32 * NB] = top;
            p[32 * NB + 1] = sum;
        }
        return;
    }
    const bool none = top == -__builtin_inff() && sum == 0.0f;
    const float inverse = none ? 0.0f : 1.0f / sum;
    const uint64_t to = token * a.ldo + static_cast<uint64_t>(head) * a.cache.dim;
    by_device_type(a.out_type, [&](auto ty) {
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t first = 32 * c + 2 * e + 4 * half;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = none ? 0.0f : o[c][e + k] * inverse;
                store4<decltype(ty)::value>(a.out, to + first, first < a.cache.dim ? a.cache.dim - first : 0u, v);
            }
    });
    if (half == 0 && a.lse != nullptr)
        a.lse[token * heads * a.group + head] = none ? top : (top + __log2f(sum)) * 0.6931471805599453f;
}

}  // namespace

void launch_kv4_prompt(const AttentionArgs &a, int depth, uint64_t tiles, hipStream_t stream) {
    const unsigned groups = static_cast<unsigned>(tiles * a.cache.heads * a.each);  // checked with the sizes
    const uint32_t n = static_cast<uint32_t>(tiles);
    by_blocks(a.cache.blocks, [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        if (depth == 1) kv4_prompt_kernel<NB, 1><<<groups, kThreads, 0, stream>>>(a, n);
        else if (depth == 2) kv4_prompt_kernel<NB, 2><<<groups, kThreads, 0, stream>>>(a, n);
        else kv4_prompt_kernel<NB, 3><<<groups, kThreads, 0, stream>>>(a, n);
    });
    BSQ_HIP(hipGetLastError());
}

}  // namespace bsq
