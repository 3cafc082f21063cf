// Attention over the paged MX4 cache (kv4_attention.hpp): the entry point, and the
// join of split tiles.
#include "kv4_attention.hpp"

#include <algorithm>
#include <cmath>

namespace bsq {
namespace {

// A wave a row of a split tile; kAtOnce parts are asked for together.
template <int NB, uint32_t kAtOnce>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttentionArgs a, uint32_t part_rows) {
    const Split s = a.splits[blockIdx.x];
    const uint32_t n_row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (s.parts == 0 || n_row >= s.rows) return;
    const auto part = [&](uint32_t b) {
        const uint64_t number = b == 0 ? s.first : s.next + static_cast<uint64_t>(b - 1) * s.step;
        return a.parts + (number * part_rows + n_row) * part_row(NB);
    };
    // lanes: parts beside one another, eight channels each; in one pass, so that a
    // part's reference and its sums are waited for together.  Four parts at once where
    // tiles have many (32 of 8 requests of 40 to 90 thousand keys: 6.5 us, one by one
    // 9.3), one where they have few (two of a chunk's tile: 19 us, with four 24).
    constexpr uint32_t kEights = 4 * NB, kBeside = NB <= 1 ? 16 : NB == 2 ? 8 : NB <= 4 ? 4 : 2;
    const uint32_t e = lane % (64 / kBeside), beside = lane / (64 / kBeside);
    float top = -__builtin_inff(), all = 0.0f, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const auto add = [&](float their_top, float their_all, const float their[8]) {
        // without a reference there are zeros, or NaN
        const float now = fmaxf(top, their_top);
        const float keep = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
        const float take = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(their_top - now);
        all = all * keep + their_all * take;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * keep + their[i] * take;
        top = now;
    };
    if (e < kEights)
        for (uint32_t b0 = beside; b0 < s.parts; b0 += kAtOnce * kBeside) {
            float x[kAtOnce][8], tops[kAtOnce], sums[kAtOnce];
#pragma unroll
            for (uint32_t n = 0; n < kAtOnce; ++n) {
                const float *p = part(min(b0 + n * kBeside, s.parts - 1));
                __builtin_memcpy(x[n], __builtin_assume_aligned(p + e * 8, 16), 32);
                tops[n] = p[32 * NB], sums[n] = p[32 * NB + 1];
            }
#pragma unroll
            for (uint32_t n = 0; n < kAtOnce; ++n)
                if (b0 + n * kBeside < s.parts) add(tops[n], sums[n], x[n]);
        }
#pragma unroll
    for (uint32_t d = 64 / kBeside; d < 64; d <<= 1) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __shfl_xor(v[i], d);
        add(__shfl_xor(top, d), __shfl_xor(all, d), x);
    }
    if (beside != 0 || e >= kEights) return;
    const uint32_t row = s.row0 + n_row;
    write_row(a, static_cast<uint64_t>(s.first_token) + row / a.group, s.head * a.group + row % a.group, e * 8, v, all, top);
}

// Requests of more rows than this are a prompt's: 16 rows a tile read and convert
// the keys once for each tile, 128 rows once for them all, by fewer waves.  16, 32,
// 48, 64 and 96 rows a request, 8 heads of 128, the one kernel against the other:
// BF16, 64 requests of 4096 keys 78, 112, 176, 176, 280 us against 175, 175, 176, 177,
// 181; 16 of 800 18, 23, 26, 29, 35 against 40 to 41; 4 of 32768 51, 65, 83, 103, 143
// against 112, 128, 129, 130, 148.  FP32, 64 of 4096: 93, 150, 221, 251, 391 against
// 407 to 415.
constexpr uint32_t kFewRows = 64;

struct Plan {
    uint32_t few;               // AttentionArgs' own
    uint32_t span = 5;          // AttentionArgs' own
    uint32_t waves = 0;         // of the kernel of few queries
    uint64_t tiles = 0;         // of the prompts' kernel
    uint32_t each = 1;
    uint64_t splits = 0, parts_bytes = 0, bytes = 0;
};
void check_sizes(const Kv4Cache &c, uint32_t width, uint32_t requests, uint64_t tokens, uint32_t q_heads) {
    BSQ_REQUIRE(q_heads >= 1 && q_heads % c.heads == 0, "kv4 attention: query heads are a multiple of the cache's");
    BSQ_REQUIRE(q_heads <= 65535, "kv4 attention: up to 65535 query heads");
    BSQ_REQUIRE(tokens <= 0x7FFFFFFFull && tokens * (q_heads / c.heads) <= 0x7FFFFFFFull, "kv4 attention: too many queries");
    BSQ_REQUIRE(requests <= 1u << 20, "kv4 attention: up to 2^20 requests");
    BSQ_REQUIRE(static_cast<uint64_t>(width) << c.shift <= 0x7FFFFFFFull - kStep, "kv4 attention: rows of the table are too long");
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
        static_assert(kStep == 1u << 5);
        const auto units_of = [&] { return (keys >> p.span) + 2 + kExtra; };
        while (tiles * units_of() >= 1ull << 31 && p.span < 30) ++p.span;
        const uint64_t units = units_of();
        BSQ_REQUIRE(tiles * units < 1ull << 31, "kv4 attention: too many queries");
        p.waves = static_cast<uint32_t>(std::min<uint64_t>(2ull * kFewWaves * cu_count(), tiles * units));
        p.splits = p.waves;
        parts = static_cast<uint64_t>(p.waves) * 2 * kTileRows;
    }
    if (prompts) {
        p.tiles = rows / kPromptRows + std::min<uint64_t>(some, ceil_div(rows, p.few + 1));
        grid_of(p.tiles * c.heads, kPromptThreads, "kv4 attention: too many queries");
        // Two workgroups of a CU run at once; up to four are made, as tiles have keys
        // of their own numbers (5 chunks of 500 tokens over 500 to 8000 keys in 400
        // tiles: 197 us with each tile whole, 171 in halves, 174 in quarters; 2048
        // tiles of a prompt 639 whole and 758 in halves).  A share has at least 1024
        // keys.
        const uint64_t shares = 4ull * cu_count() / (p.tiles * c.heads);
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

template <int NB, uint32_t kAtOnce>
void join(const AttentionArgs &a, uint64_t splits, uint32_t part_rows, uint64_t rows, hipStream_t s) {
    rows = std::min<uint64_t>(rows, part_rows);
    kv4_join_kernel<NB, kAtOnce><<<dim3(static_cast<unsigned>(splits), static_cast<unsigned>((rows + 3) / 4)), 256, 0, s>>>(a, part_rows);
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
        const float factor = static_cast<float>(std::fabs(static_cast<double>(scale)) * 1.44269504088896340736);
        BSQ_REQUIRE(std::isfinite(factor), "kv4 attention: the scale is too large");
        BSQ_REQUIRE(causal == 0 || causal == 1, "kv4 attention: causal is 0 or 1");
        BSQ_REQUIRE(causal == 1 || window == 0, "kv4 attention: a window is of causal attention");
        BSQ_REQUIRE(d_starts != nullptr || tokens == requests, "kv4 attention: without starts each request has one query");
        if (!some) return;
        BSQ_REQUIRE(d_lengths != nullptr && (width == 0 || d_table != nullptr), "kv4 attention: null argument");
        check_dense(d_q, tq, "kv4 attention: null queries");
        check_dense(d_out, to, "kv4 attention: null output");
        // others may still read queries where a tile's results are written
        BSQ_REQUIRE(!overlap(tokens, CallRows(d_q, ldq, row, tq), CallRows(d_out, ldo, row, to)), "kv4 attention: out overlaps the queries");
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
        a.factor = factor;
        a.negate = scale < 0.0f;
        a.causal = causal != 0;
        a.window = window >= static_cast<uint64_t>(width) << a.cache.shift ? 0u : window;  // all of a request's
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
            if (p.waves > 0) {
                if (depth == 1) launch_kv4_few<1>(a, p.waves, s);
                else if (depth == 2) launch_kv4_few<2>(a, p.waves, s);
                else launch_kv4_few<3>(a, p.waves, s);
                if (p.waves > 1) join<NB, 4>(a, p.waves, kTileRows, rows, s);
            }
            if (p.tiles > 0) {
                launch_kv4_prompt(a, depth, p.tiles, s);
                if (p.each > 1) join<NB, 1>(a, p.tiles * a.cache.heads, kPromptRows, rows, s);
            }
        });
    });
}

}  // extern "C"
