// The paged cache of keys and values in MX4: its layout and what its kernels
// share (kv4.hip, kv4_attention.hip).
//
// Page p, head h: a run of bytes at (p * heads + h) * head_bytes that holds the
// keys' codes, the values' codes, the keys' scales, the values' scales.  Codes
// are row-major, so that a token's are whole words that its own append writes;
// scales of 16 tokens lie together as [token % 4][block][token / 4], the order in
// which a lane of the attention's matrix instructions takes its tokens: the four
// that it needs of a block are one word.
#pragma once

#include "mx4.hpp"

#include "bitsqz_llm_c.h"

namespace bsq {

constexpr uint32_t kKv4MaxDim = 256;

struct Kv4Cache {
    uint8_t *pages;
    uint32_t head_bytes;  // of a page fewer than 2^31
    uint32_t count, shift, heads, dim, blocks;  // a page has 1 << shift tokens

    __host__ __device__ uint32_t page() const { return 1u << shift; }
    __host__ __device__ uint32_t row_bytes() const { return blocks * 16; }
    __device__ __forceinline__ uint8_t *head(uint32_t page_number, uint32_t h) const {
        return pages + static_cast<uint64_t>(page_number) * (heads * head_bytes) + h * head_bytes;
    }
    // from a head's bytes: the codes and the scale byte of block b of token t
    // (in the page) of the keys (0) or values (1)
    __device__ __forceinline__ uint64_t codes_at(uint32_t which, uint32_t t) const {
        return static_cast<uint64_t>((which << shift) + t) * row_bytes();
    }
    __device__ __forceinline__ uint64_t scale_at(uint32_t which, uint32_t t, uint32_t b) const {
        return (static_cast<uint64_t>(2 * row_bytes()) << shift) + (static_cast<uint64_t>(which * blocks) << shift) +
               (t >> 4) * 16 * blocks + 4 * ((t & 3) * blocks + b) + ((t >> 2) & 3);
    }
};

inline Kv4Cache kv4_cache(const bsq_kv4_cache_t *c, bool followed = true) {
    BSQ_REQUIRE(c != nullptr, "kv4: null cache");
    uint32_t shift = 4;
    while (shift < 8 && (1u << shift) != c->page) ++shift;
    BSQ_REQUIRE((1u << shift) == c->page, "kv4: a page has 16, 32, 64, 128 or 256 tokens");
    BSQ_REQUIRE(c->dim >= 1 && c->dim <= kKv4MaxDim, "kv4: heads of 1 to 256 values");
    BSQ_REQUIRE(c->heads >= 1 && c->heads <= 65535, "kv4: 1 to 65535 heads");
    BSQ_REQUIRE(c->pages <= 0x7FFFFFFFull >> shift, "kv4: too many pages");
    if (followed) {
        BSQ_REQUIRE(c->pages >= 1 && c->d_pages != nullptr, "kv4: null cache");
        BSQ_REQUIRE((reinterpret_cast<uintptr_t>(c->d_pages) & 15) == 0, "kv4: pages are 16-byte aligned");
    }
    const uint32_t blocks = static_cast<uint32_t>(ceil_div(c->dim, kMx4Block));
    const uint64_t head_bytes = static_cast<uint64_t>(34 * blocks) << shift;
    BSQ_REQUIRE(head_bytes * c->heads <= 0x7FFFFFFFull, "kv4: a page has 2^31 bytes or more");
    return {c->d_pages, static_cast<uint32_t>(head_bytes), static_cast<uint32_t>(c->pages), shift, c->heads,
            c->dim, blocks};
}

// A call's rows: `bytes` each, `pitch` bytes apart.
struct CallRows {
    uintptr_t at;
    uint64_t pitch, bytes;
    CallRows(const void *p, uint64_t ld, uint64_t width, Mx4Type t)
        : at(reinterpret_cast<uintptr_t>(p)), pitch(ld * type_bytes(t)), bytes(width * type_bytes(t)) {}
};
// Whether rows of two kinds, `tokens` of either, share a byte.  Of one pitch they may
// lie side by side; of two they count as sharing one wherever their spans cross.
inline bool overlap(uint64_t tokens, const CallRows &a, const CallRows &b) {
    const uint64_t a_span = (tokens - 1) * a.pitch + a.bytes, b_span = (tokens - 1) * b.pitch + b.bytes;
    if (a.at >= b.at + b_span || b.at >= a.at + a_span) return false;
    if (a.pitch != b.pitch) return true;
    const CallRows &low = a.at <= b.at ? a : b, &high = a.at <= b.at ? b : a;
    const uint64_t on = (high.at - low.at) % low.pitch;  // bytes from a row of `low` to one of `high`
    return on < low.bytes || on + high.bytes > low.pitch;
}

}  // namespace bsq
