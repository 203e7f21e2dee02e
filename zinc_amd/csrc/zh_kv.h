// zh_kv.h — what the batched operators over a paged cache share (zh_kv.hip,
// zh_shared_attn.hip).
#pragma once
#include <algorithm>

#include "zh_internal.h"

static inline bool kv_in_range(const zh_buf *b, uint64_t off, uint64_t n) {
    return b && off <= b->size && n <= b->size - off;
}
bool kv_batch_ok(const zh_kv_batch *kv);
// Byte ranges [a0, a0 + an) of a and [b0, b0 + bn) of b share a byte.
bool kv_rows_overlap(const zh_buf *a, uint64_t a0, uint64_t an, const zh_buf *b, uint64_t b0, uint64_t bn);
// Two sets of rows of one stride (elements of `size` bytes) whose byte ranges
// overlap: whether their columns are apart (parts of one stacked matrix).
static inline bool kv_columns_apart(const zh_buf *a, uint64_t a_off, const zh_buf *b, uint64_t b_off, uint64_t stride,
                                    uint64_t a_width, uint64_t b_width, uint32_t size) {
    const uint64_t pa = (uint64_t)(uintptr_t)a->ptr + a_off, pb = (uint64_t)(uintptr_t)b->ptr + b_off;
    const uint64_t row = stride * size, d = pb >= pa ? (pb - pa) % row : (row - (pa - pb) % row) % row;
    // b's columns start d bytes after a's: past a's, and not into a's next row
    return d >= a_width * size && d + b_width * size <= row;
}
// Cache slot (token index) of position pos of sequence s; false: outside the
// tables or the cache. (The page entry is compared, not its token, which an
// entry from 2^28 on would wrap.)
__host__ __device__ __forceinline__ bool kv_slot(const uint32_t *tables, uint32_t n_seq, uint32_t stride,
                                                 uint32_t cache_tokens, uint32_t s, uint32_t pos, uint32_t &slot) {
    if (s >= n_seq || pos / 16 >= stride) return false;
    const uint32_t page = tables[(size_t)s * stride + pos / 16];
    if (page >= cache_tokens / 16) return false;
    slot = page * 16 + pos % 16;
    return true;
}
