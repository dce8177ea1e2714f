// kv8_index.h -- the index arithmetic of the 8-bit paged cache, for the kernels and for host
// tests.  Nothing read from device memory (row bounds, slots, positions, page ids) is trusted:
// every value passes one of these functions before it becomes an address.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "../../include/mossgpu.h"
#include "op_support.h"

#if defined(__CUDACC__)
#define MOSSGPU_HD __host__ __device__ __forceinline__
#else
#define MOSSGPU_HD inline
#endif

namespace mossgpu {

constexpr int kKv8Page = 16;  // positions per page, as in the fp16 cache

// Sequence s's new rows, clamped into [0, rows]: rows r0 <= r < r1.
struct RowRange {
    int r0, r1;
};
MOSSGPU_HD RowRange kv8_rows(int start, int end, int rows) {
    RowRange r;
    r.r0 = start < 0 ? 0 : start > rows ? rows : start;
    r.r1 = end < r.r0 ? r.r0 : end > rows ? rows : end;
    return r;
}

// Positions slot `slot` can hold, 0 for a slot outside the table.
MOSSGPU_HD int kv8_capacity(const mossgpu_kv8_cache &c, int slot) {
    return slot < 0 || slot >= c.n_slots ? 0 : c.pages_per_slot * kKv8Page;
}

// Positions of a sequence that exist: its context and its new rows as far as the slot's pages
// reach.  *status gets kStatusBadPosition where they do not reach, or the context is negative.
struct SeqSpan {
    int ctx, total;
};
MOSSGPU_HD SeqSpan kv8_span(const mossgpu_kv8_cache &c, int slot, int ctx, int new_rows, int *status) {
    SeqSpan s;
    s.ctx = s.total = 0;
    const int cap = kv8_capacity(c, slot);
    if (ctx < 0 || ctx > cap || new_rows > cap - ctx) *status = kStatusBadPosition;
    if (ctx < 0) return s;
    s.ctx = ctx < cap ? ctx : cap;
    s.total = new_rows > cap - s.ctx ? cap : s.ctx + new_rows;
    return s;
}

// A page id as it stands in the table, or -1 (and *status) outside the pool.
MOSSGPU_HD int kv8_page(const mossgpu_kv8_cache &c, int page, int *status) {
    if (page >= 0 && page < c.n_pages) return page;
    *status = kStatusBadPage;
    return -1;
}

// Attention's plan counts tiles in 32 bits.  Row bounds that ascend keep a call's sum below kKv8MaxTiles, which the
// host checks; bounds that do not (a row may then belong to many sequences) can pass it, so every sum stops there
// instead of wrapping, and a plan that gets there is none.
constexpr uint32_t kKv8MaxTiles = 0x7fffffffu;
MOSSGPU_HD uint32_t kv8_add_tiles(uint32_t a, uint32_t b) {  // both at most kKv8MaxTiles
    const uint32_t s = a + b;
    return s < kKv8MaxTiles ? s : kKv8MaxTiles;
}
// Tiles of a sequence, `tiles` for each block of block_rows of its new rows times the heads of a group (at most 2^30).
MOSSGPU_HD uint32_t kv8_seq_tiles(uint32_t tiles, int new_rows, int group, int block_rows) {
    const uint64_t n = uint64_t(tiles) * uint32_t((new_rows * group + block_rows - 1) / block_rows);
    return n < kKv8MaxTiles ? uint32_t(n) : kKv8MaxTiles;
}

// Element offsets: codes [n_pages][2][kv_heads][16][head_dim], scales [n_pages][2][kv_heads][16].
MOSSGPU_HD size_t kv8_cell(const mossgpu_kv8_cache &c, int page, int half, int head, int off) {
    return ((size_t(page) * 2 + size_t(half)) * size_t(c.kv_heads) + size_t(head)) * kKv8Page + size_t(off);
}

}  // namespace mossgpu
