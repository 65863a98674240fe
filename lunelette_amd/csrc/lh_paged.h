// The paged KV cache on the device: page layout and the sequences of a call.
#pragma once

#include "lh_device.h"
#include "lh_serving.h"

namespace lh {

// A page holds its KV heads one after another, a head's part the keys' codes,
// the values' codes and (Q4) a word per key and a word per value with the BF16
// scale below and the zero above. Codes are FP16 values or nibbles, in the order
// in which the attention's 16x16x32 matrix instructions take them:
// - keys: tiles of 16 positions. Lane l = 16 g + r of a wave has position r's
//   dims 32 j + 8 g .. + 7 for every j, F16 as tile [j][lane][8], Q4 as a word
//   per j, [lane][j];
// - values: blocks of 32 positions. Lane 16 g + r has dim 16 i + r of positions
//   4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 for every 16-dim tile i, F16 as block
//   [i][lane][8], Q4 as a word per i, [i / 4][lane][i % 4].
// Eight codes in a word: the element 2 n in nibble n, 2 n + 1 in nibble 4 + n.
template <int D, bool Q4>
struct PageLayout {
    static constexpr uint32_t vector = Q4 ? D / 2 : 2 * D;   // bytes of a vector's codes

    __device__ static __forceinline__ size_t head_bytes(uint32_t page_size)
    {
        return (size_t)page_size * (2 * vector + (Q4 ? 8 : 0));
    }
    // Byte offsets in a head's part. slot: position in the page.
    __device__ static __forceinline__ uint32_t values(uint32_t page_size)
    {
        return page_size * vector;
    }
    __device__ static __forceinline__ uint32_t scales(uint32_t page_size, int which)
    {
        return page_size * (2 * vector + 4 * which);
    }
    // The 8 codes of dims 8 c .. 8 c + 7 of a key (4 bytes or 16).
    __device__ static __forceinline__ uint32_t key_chunk(uint32_t slot, uint32_t c)
    {
        const uint32_t tile = slot >> 4, lane = 16 * (c & 3) + (slot & 15), j = c >> 2;
        return Q4 ? tile * 16 * vector + lane * (D / 8) + j * 4
                  : tile * 16 * vector + j * 1024 + lane * 16;
    }
    // The 8 codes of dim d of the values at 32 * (slot / 32) + 4 g + {0..3, 16..19}.
    __device__ static __forceinline__ uint32_t value_chunk(uint32_t slot, uint32_t d, uint32_t g)
    {
        const uint32_t block = slot >> 5, lane = 16 * g + (d & 15), i = d >> 4;
        return block * 32 * vector + (Q4 ? (i >> 2) * 1024 + lane * 16 + (i & 3) * 4
                                         : i * 1024 + lane * 16);
    }
};

// Nibble shift of element e of a word.
__device__ __forceinline__ uint32_t nibble_at(uint32_t e)
{
    return 4 * (e >> 1) + 16 * (e & 1);
}

struct Pages {
    uint8_t* base;
    uint32_t kv_heads, page_size, pages;
};

struct Batch {
    const int32_t *query_start, *length, *table;
    uint32_t tokens, width;
};

// Rows [begin, begin + count) of sequence s at positions first .. first + count - 1
// (first may be negative). The device arrays are not trusted further than that:
// rows stay inside the call's tensors whatever they hold.
struct Span {
    int64_t begin, count, first;
};

__device__ __forceinline__ Span batch_span(const Batch& b, uint32_t s)
{
    const int64_t limit = b.tokens;
    int64_t begin = b.query_start[s], end = b.query_start[s + 1];
    begin = begin < 0 ? 0 : begin > limit ? limit : begin;
    end = end < begin ? begin : end > limit ? limit : end;
    return {begin, end - begin, (int64_t)b.length[s] - (end - begin)};
}

// The part of KV head h in the page of position p (any position of its 32-position
// block does), or NULL when the position has no place.
template <int D, bool Q4>
__device__ __forceinline__ uint8_t* page_part(const Pages& c, const Batch& b, uint32_t s,
    int64_t p, uint32_t h)
{
    if (p < 0) {
        return nullptr;
    }
    const int64_t at = p / c.page_size;
    if (at >= b.width) {
        return nullptr;
    }
    const int32_t id = b.table[(size_t)s * b.width + at];
    if (id < 0 || (uint32_t)id >= c.pages) {
        return nullptr;
    }
    return c.base + ((size_t)id * c.kv_heads + h) * PageLayout<D, Q4>::head_bytes(c.page_size);
}

static inline Pages pages_of(const lh_paged_cache* c)
{
    return {static_cast<uint8_t*>(c->d_pages), c->kv_heads, c->page_size, c->pages};
}

static inline Batch batch_of(const lh_paged_batch* b)
{
    return {b->d_query_start, b->d_length, b->d_table, b->tokens, b->table_width};
}

// Calls f<D, Q4>() for the cache's head size and kind.
#define LH_FOR_CACHE(cache, f, ...) \
    ((cache)->head_dim == 64 ? ((cache)->kind == LH_CACHE_Q4 ? f<64, true>(__VA_ARGS__) \
            : f<64, false>(__VA_ARGS__)) \
        : ((cache)->kind == LH_CACHE_Q4 ? f<128, true>(__VA_ARGS__) : f<128, false>(__VA_ARGS__)))

}  // namespace lh
