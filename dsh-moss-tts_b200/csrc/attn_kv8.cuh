// attn_kv8.cuh -- attention of one or a few new rows a sequence over the 8-bit paged cache.
//
// DIRECT: a CTA has a whole unit, its warps the tiles in turn; no plan, no second launch.
//
// Work otherwise.  A unit is (sequence, kv head, block of query rows); its rows are the sequence's
// new rows times the query heads of the group, so a cache byte serves all of them.  A unit's
// positions come in tiles of 32 (two pages).  All tiles of one head, in order, are cut into equal
// runs, one run of one head per warp of the grid: however ragged the batch is, every warp has the
// same work.  The heads of a run go to neighbouring warps, since a page's heads lie side by side (512
// long sequences: with the runs of a head behind one another 2% more time).  A warp that has a whole
// unit writes its rows; a unit cut between warps leaves partial sums in the workspace, which k_attn_kv8_join (a
// dependent launch) merges in a fixed order, so that a result does not depend on timing.
//
// A tile.  K, V and their scales of the pages (each contiguous) are copied to a stage of the warp's own
// ring in shared memory, 16 bytes a lane (with bulk copies of 1 KB, which are issued one lane after the
// other, those sequences take 7% more).  No barrier but the warp's own.  S = q K^T
// and o += w V are mma.sync m16n8k16 products in fp16, in which every 8-bit code is exact.  Which
// element of the head dimension is the k-th of a product, and which position is the n-th, is free as
// long as both operands agree.  Here a lane takes 16 consecutive codes of a K row, the same columns of
// four neighbouring V rows, and those four positions' scales as one vector, so that codes go from
// shared memory to a fragment by wide loads and conversions alone.  The scales of a position multiply
// its score (K) and its weight (V) in fp32.
//
// Precision.  A query row is scaled by a power of two to [128, 256) and rounded to fp16, exact for
// bf16 and fp16 inputs.  Weights are w = 2^(rf (s - m) + 140 - E) sv, s the scores without the row's factor rf, m
// their running maximum and E the exponent of the largest V scale that the row has seen: w < 2^14 fits fp16
// whatever the scales are, and, since the difference comes before the factor, however large the scores are.
// For bf16 outputs w is rounded to fp16 (2^-11 against the output's 2^-8), 16 rows a product.  For fp32 and
// fp16 outputs q and w are split into an upper and a lower
// fp16 part (22 bits) that occupy rows g and g + 8 of the same product, 8 rows a product; since the
// tensor cores truncate when they accumulate, such products start from zero every tile and are added
// in fp32.  Statistics, sums and partials are fp32.
//
// Measured on one B200: 512 sequences of 256-4096 positions, 12 heads of 64, int8: 301 us (6.0 TB/s, 92%
// of the measured copy rate) in bursts of 20 calls, 318-345 us (81-87%, by card) when repeated for seconds, as the
// card then lowers its clocks: about 455 instructions a tile of 32 positions keep the schedulers 62% busy.
#pragma once

#include <float.h>

#include <type_traits>

#include "f32x2.cuh"
#include "rope_kv8.cuh"

namespace mossgpu {

constexpr int kAk8MaxSeqs = 4096;
constexpr int kAk8Tile = 32;  // positions: two pages

template <int D>
struct Ak8Shape {
    static constexpr int kBlock = 16 * D;                      // bytes of one page's K (or V) of a head
    static constexpr int kStage = 4 * kBlock + 4 * 64;         // K, V of two pages, then their scales
    static constexpr int kWarps = D == 64 ? 16 : 12;
    static constexpr int kStages = D == 64 ? 3 : 2;
    static constexpr int kRing = kStage * kStages * kWarps;    // 208,896 and 202,752 bytes
};

// k_attn_kv8_few: pages of a tile, warps of a CTA, stages of a warp's ring
template <int D>
struct Ak8Few {
    static constexpr int kPages = 2;
    static constexpr int kBlock = 16 * D;
    static constexpr int kStage = kPages * (2 * kBlock + 128);
    static constexpr int kWarps = D == 64 ? 16 : 12;
    static constexpr int kStages = D == 64 ? 3 : 2;
    static constexpr int kRing = kStage * kStages * kWarps;
};

struct AttnKv8 {
    mossgpu_kv8_cache cache;
    mossgpu_seq_batch seqs;
    mossgpu_attention_kv8_args a;
    int group;       // query heads per kv head
    int runs;        // most runs a head's tiles are cut into: runs * kv_heads <= warps of the grid
    int tile_rows;   // rows of a unit
    int part_rows;   // rows a partial keeps
    int vec_q, vec_out;
    uint32_t *plan;  // [n_seqs + 1] tiles (over row blocks, per kv head) before a sequence; then [n_seqs] tiles of one block
    float *part;     // [2 * runs * kv_heads][part_rows][head_dim + 4]: sums, then their reference and l
    int *status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Copies NP pages of a head (id: lane i < NP has page i's, -1 for none) to a stage:
// K pages, V pages, then the scales as [k, v][page][16].
template <int D, int NP>
__device__ __forceinline__ void copy_pages(const mossgpu_kv8_cache &c, int head, uint32_t dst, int id) {
    constexpr int kBlock = 16 * D;
    const int lane = threadIdx.x & 31;
    const uint32_t page_bytes = uint32_t(2 * kBlock) * uint32_t(c.kv_heads);
#pragma unroll
    for (int pg = 0; pg < NP; ++pg) {
        const int page = __shfl_sync(0xffffffffu, id, pg);
        if (page >= 0) {
            const uint8_t *k = static_cast<const uint8_t *>(c.codes) + uint64_t(uint32_t(page)) * page_bytes + uint32_t(head * kBlock + lane * 16);
            const uint8_t *v = k + page_bytes / 2;
#pragma unroll
            for (int i = 0; i < kBlock / 512; ++i) {
                cp_async16(dst + pg * kBlock + lane * 16 + i * 512, k + i * 512);
                cp_async16(dst + (NP + pg) * kBlock + lane * 16 + i * 512, v + i * 512);
            }
        }
    }
    // lane: K or V (lane / (4 NP)), page (lane / 4), 4 scales
    const int page = __shfl_sync(0xffffffffu, id, (lane >> 2) & (NP - 1));
    if (lane < 8 * NP && page >= 0) {
        const float *s = c.scales + uint64_t(uint32_t(page)) * uint32_t(2 * kKv8Page * c.kv_heads) +
                         uint32_t(((lane >= 4 * NP ? c.kv_heads : 0) + head) * kKv8Page + (lane & 3) * 4);
        cp_async16(dst + 2 * NP * kBlock + lane * 16, s);
    }
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same from zero
__device__ __forceinline__ void mma16816_0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                           uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ uint32_t pack2(float2 x) { return half2_bits(__float22half2_rn(x)); }
// the fp16 parts of a pair: upper returned, lower = what the upper leaves
__device__ __forceinline__ uint32_t split2(float2 x, uint32_t *lower) {
    const __half2 h = __float22half2_rn(x);
    const float2 f = __half22float2(h);
    *lower = pack2(make_float2(x.x - f.x, x.y - f.y));
    return half2_bits(h);
}

// Codes 0, 1 (lo) and 2, 3 (hi) of a word as fp16 pairs.
template <int FORMAT>
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (FORMAT == MOSSGPU_KV_INT8) {
        // code + 128 behind the fp16 exponent of 1024; the subtraction is exact
        const uint32_t b = w ^ 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
        uint32_t l = __byte_perm(b, 0x64646464u, 0x4140), h = __byte_perm(b, 0x64646464u, 0x4342);
        lo = half2_bits(__hsub2(*reinterpret_cast<__half2 *>(&l), off));
        hi = half2_bits(__hsub2(*reinterpret_cast<__half2 *>(&h), off));
    } else {
        asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// A query row whose largest element is `top` enters the products times `to`, a power of two with the sign of the
// scale that takes it to [128, 256) (elements below 2^-119 stay below that), and its products with K times `rf` are
// scores in log2.  rf is finite and above 0, as 0 and infinity would make NaN of scores that are masked or 0.
__device__ __forceinline__ void query_factors(float top, float scale, float &to, float &rf) {
    const int e = max(-119, int(__float_as_uint(top) >> 23) - 127);  // 128 for infinity and NaN: `to` is still a number
    to = scale == 0.f ? 0.f : copysignf(pow2i(7 - e), scale);
    rf = scale == 0.f ? 1.f : fminf(fmaxf(fabsf(scale) * pow2i(e - 7) * 1.4426950408889634f, __int_as_float(1)), FLT_MAX);
}

// What scores are taken relative to, where their running maximum is m
__device__ __forceinline__ float score_base(float m) { return m == -INFINITY ? 0.f : m; }
// What earlier sums are multiplied by when the maximum goes from m0 to m and the V scales' exponent from E0 to E
__device__ __forceinline__ float sums_factor(float m0, float m, float rf, float E0, float E) { return ex2(fmaf(m0 - score_base(m), rf, E0 - E)); }
// Partial sums are kept relative to their maximum, which is stored in log2 (finite where there is any), and 2^-20, so
// that a million positions' values of any size add up: sums relative to `bias` - E times this
__device__ __forceinline__ float part_factor(float E, int bias) { return pow2i(int(E) - bias - 20); }
__device__ __forceinline__ float part_reference(float m, float rf) { return m == -INFINITY ? m : fmaxf(fminf(m * rf, 0.5f * FLT_MAX), -0.5f * FLT_MAX); }

// The bits of a scale's size, 0 for infinity and NaN
__device__ __forceinline__ uint32_t finite_bits(float scale) {
    const uint32_t b = __float_as_uint(scale) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// 8 elements of a row of q, whatever its type
__device__ __forceinline__ void load_q8(const void *q, int type, bool vec, int64_t at, float (&x)[8]) {
    if (type == MOSSGPU_F32)
        load8(static_cast<const float *>(q) + at, vec, x);
    else if (type == MOSSGPU_F16)
        load8(static_cast<const __half *>(q) + at, vec, x);
    else
        load8(static_cast<const __nv_bfloat16 *>(q) + at, vec, x);
}
__device__ __forceinline__ float2 load_q2(const void *q, int type, int64_t at) {
    if (type == MOSSGPU_F32) {
        const float *x = static_cast<const float *>(q) + at;
        return make_float2(x[0], x[1]);
    }
    if (type == MOSSGPU_F16) {
        const __half *x = static_cast<const __half *>(q) + at;
        return make_float2(__half2float(x[0]), __half2float(x[1]));
    }
    const __nv_bfloat16 *x = static_cast<const __nv_bfloat16 *>(q) + at;
    return make_float2(__bfloat162float(x[0]), __bfloat162float(x[1]));
}
__device__ __forceinline__ void store_out8(void *o, int type, bool vec, int64_t at, const float (&x)[8]) {
    if (type == MOSSGPU_F32)
        store8(static_cast<float *>(o) + at, vec, x);
    else if (type == MOSSGPU_F16)
        store8(static_cast<__half *>(o) + at, vec, x);
    else
        store8(static_cast<__nv_bfloat16 *>(o) + at, vec, x);
}

// Run r of n has the tiles [total r / n, total (r + 1) / n); n <= total.
__device__ __forceinline__ int64_t run_begin(int64_t total, int n, int r) { return total * r / n; }
__device__ __forceinline__ int run_of(int64_t total, int n, int64_t g) { return int(((g + 1) * n - 1) / total); }
__device__ __forceinline__ int runs_used(int64_t total, int runs) { return int(total < runs ? total : runs); }

// Tiles (of TILE positions, over blocks of ROWS query rows, per kv head) before each sequence, in
// shared memory, and, from CTA 0, in the workspace for k_attn_kv8_join.  Returns those of the batch, 0 where row
// bounds that do not ascend make them too many to count.
template <int ROWS, int TILE, int WARPS>
__device__ __forceinline__ int64_t plan_tiles(const AttnKv8 &p, uint32_t *plan) {
    __shared__ uint32_t warp_sum[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_seqs = p.seqs.n_seqs;
    uint32_t before = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += WARPS * 32) {
        const int s = s0 + int(threadIdx.x);
        uint32_t mine = 0;
        if (s < n_seqs) {
            const RowRange r = kv8_rows(__ldg(p.seqs.row_start + s), __ldg(p.seqs.row_start + s + 1), p.seqs.rows);
            const int slot = __ldg(p.seqs.slot + s), ctx = __ldg(p.seqs.ctx_len + s);
            int status = 0;
            if (r.r1 > r.r0) {
                const SeqSpan span = kv8_span(p.cache, slot, ctx, r.r1 - r.r0, &status);
                const uint32_t tiles = span.total > 0 ? (span.total + TILE - 1) / TILE : 1;
                mine = kv8_seq_tiles(tiles, r.r1 - r.r0, p.group, ROWS);
                if (blockIdx.x == 0) p.plan[n_seqs + 1 + s] = tiles;
            }
            if (blockIdx.x == 0) op_report(p.status, status);
        }
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = kv8_add_tiles(sum, v);
        }
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        uint32_t base = before, all = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) base = kv8_add_tiles(base, warp_sum[w]);
            all = kv8_add_tiles(all, warp_sum[w]);
        }
        if (s < n_seqs) plan[s] = kv8_add_tiles(base, sum) - mine;
        before = kv8_add_tiles(before, all);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (before == kKv8MaxTiles) {
            before = 0;
            if (blockIdx.x == 0) op_report(p.status, kStatusBadPosition);
        }
        plan[n_seqs] = before;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s <= n_seqs; s += WARPS * 32) p.plan[s] = plan[s];
    return int64_t(plan[n_seqs]);
}

// This warp's run, as tiles [g, g_end) of a head: the (run, head) pairs are dealt to the CTAs evenly and in order.
struct Run {
    int64_t g, g_end;
    int item, head;
};
template <int WARPS>
__device__ __forceinline__ bool warp_run(const AttnKv8 &p, int64_t total, Run &w) {
    const int H = p.cache.kv_heads, used = runs_used(total, p.runs);
    const int64_t items = int64_t(used) * H;
    const int lo = int(items * blockIdx.x / gridDim.x), hi = int(items * (blockIdx.x + 1) / gridDim.x);
    w.item = lo + int(threadIdx.x >> 5);
    if (w.item >= hi) return false;
    const int r = w.item / H;
    w.head = w.item - r * H;
    w.g = run_begin(total, used, r);
    w.g_end = run_begin(total, used, r + 1);
    return true;
}

// The unit that tile g of a head belongs to, and its tiles [t0, t1) in a run that ends at g_end.
struct Unit {
    RowRange rr;
    SeqSpan span;
    int head, block, tiles, t0, t1, n_rows, n_pages;
    const int32_t *table;
};
// A sequence's share of it; returns the status of its span.
__device__ __forceinline__ int fill_unit(const AttnKv8 &p, RowRange rows, int slot, int ctx, int tile, Unit &u) {
    u.rr = rows;
    int status = 0;
    u.span = kv8_span(p.cache, slot, ctx, u.rr.r1 - u.rr.r0, &status);
    u.tiles = u.span.total > 0 ? (u.span.total + tile - 1) / tile : 1;
    u.n_rows = (u.rr.r1 - u.rr.r0) * p.group;
    u.table = p.cache.page_table + size_t(u.span.total > 0 ? slot : 0) * p.cache.pages_per_slot;
    u.n_pages = (u.span.total + kKv8Page - 1) / kKv8Page;
    return status;
}
// E elements of an output row, times f
template <int E>
__device__ __forceinline__ void store_row(const AttnKv8 &p, int row, int head, int at, const float (&y)[E], float f) {
    const int64_t to = int64_t(row) * p.a.out_row_stride + int64_t(head) * p.a.out_head_stride + at;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (p.a.type == MOSSGPU_F32)
            static_cast<float *>(p.a.out)[to + i] = y[i] * f;
        else if (p.a.type == MOSSGPU_F16)
            static_cast<__half *>(p.a.out)[to + i] = __float2half_rn(y[i] * f);
        else
            static_cast<__nv_bfloat16 *>(p.a.out)[to + i] = __float2bfloat16_rn(y[i] * f);
    }
}
__device__ __forceinline__ Unit find_unit(const AttnKv8 &p, const uint32_t *plan, const Run &w, int tile) {
    int lo = 0, hi = p.seqs.n_seqs;  // the last sequence that begins at or before g: it has tiles
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(plan[mid]) <= w.g) lo = mid; else hi = mid;
    }
    Unit u;
    fill_unit(p, kv8_rows(__ldg(p.seqs.row_start + lo), __ldg(p.seqs.row_start + lo + 1), p.seqs.rows), __ldg(p.seqs.slot + lo),
              __ldg(p.seqs.ctx_len + lo), tile, u);  // its status is reported by plan_tiles
    u.head = w.head;
    const uint32_t at = uint32_t(w.g) - plan[lo];
    u.block = int(at / uint32_t(u.tiles));
    u.t0 = int(at - uint32_t(u.block) * uint32_t(u.tiles));
    u.t1 = int(min(int64_t(u.tiles), u.t0 + (w.g_end - w.g)));
    return u;
}

// Unit `index` of the batch where a CTA has a whole one: block (index / heads) of all sequences' blocks
// of ROWS query rows.  n_rows is 0 past the last.
template <int ROWS>
__device__ __forceinline__ Unit direct_unit(const AttnKv8 &p, int index, int tile, int *status) {
    const int lane = threadIdx.x & 31, H = p.cache.kv_heads, want = index / H;
    Unit u;
    u.n_rows = 0;
    int before = 0;
    for (int s0 = 0; s0 < p.seqs.n_seqs; s0 += 32) {
        int blocks = 0, slot = -1, ctx = 0;
        RowRange r{0, 0};
        if (s0 + lane < p.seqs.n_seqs) {
            r = kv8_rows(__ldg(p.seqs.row_start + s0 + lane), __ldg(p.seqs.row_start + s0 + lane + 1), p.seqs.rows);
            slot = __ldg(p.seqs.slot + s0 + lane), ctx = __ldg(p.seqs.ctx_len + s0 + lane);
            blocks = ((r.r1 - r.r0) * p.group + ROWS - 1) / ROWS;
        }
        int sum = blocks;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + sum > want);
        if (past) {
            const int at = __ffs(past) - 1;
            r.r0 = __shfl_sync(0xffffffffu, r.r0, at), r.r1 = __shfl_sync(0xffffffffu, r.r1, at);
            *status = fill_unit(p, r, __shfl_sync(0xffffffffu, slot, at), __shfl_sync(0xffffffffu, ctx, at), tile, u);
            u.head = index - want * H;
            u.block = want - before - __shfl_sync(0xffffffffu, sum - blocks, at);
            u.t0 = 0, u.t1 = u.tiles;
            return u;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return u;
}

// Where a CTA has a whole unit: its warps' sums, ROWS rows of D + 4 floats each (sums, reference, l) at `part` +
// warp * stride, to the output.
template <int D, int WARPS>
__device__ __forceinline__ void join_warps(const AttnKv8 &p, const Unit &u, int rows, const float *part, int stride) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < rows; r += WARPS) {
        const int x = u.block * p.tile_rows + r;
        if (x >= u.n_rows) break;
        const float ref = lane < WARPS ? part[lane * stride + r * (D + 4) + D] : -INFINITY;
        float top = ref;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float f = top == -INFINITY ? 0.f : ex2(ref - top);
        float l = lane < WARPS ? part[lane * stride + r * (D + 4) + D + 1] * f : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float y[E];
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = 0.f;
#pragma unroll 8
        for (int w = 0; w < WARPS; ++w) {
            const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = fmaf(part[w * stride + r * (D + 4) + lane * E + i], fw, y[i]);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store_row<E>(p, u.rr.r0 + x / p.group, u.head * p.group + x % p.group, lane * E, y, inv);
    }
}

// How a warp's rows enter the products.
constexpr int kSplit = 0;   // fp16, 8 rows as upper and lower parts: fp32 and fp16 outputs
constexpr int kHalf = 1;    // fp16, 16 rows: bf16 outputs

// A warp's rows: lane (g, t) has row g of its 8 (kSplit), or rows g and g + 8.
template <int D, int MODE>
struct Rows {
    static constexpr int NR = MODE == kSplit ? 1 : 2;  // rows of a lane
    static constexpr int NJ = D / 8;                   // output columns of a lane, per row: 2 NJ
    static constexpr int kRows = 8 * NR;
    uint32_t q[D / 16][4];
    float rf[NR];            // what makes a product a score in log2, above 0
    int new_row[NR];         // which new row of the sequence; -1: none
    float o[NJ][2 * NR], m[NR], l[NR];  // m: the largest score, without rf
    float E[NR];             // biased exponents of the largest V scales they have seen (scales below 2^-87 lose bits of their weights)
};

// The query rows from `first` on as fragments; the sign of the scale goes into them.
template <int D, int MODE>
__device__ __forceinline__ void load_rows(const AttnKv8 &p, const Unit &u, int first, Rows<D, MODE> &w) {
    const int lane = threadIdx.x & 31, row8 = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < w.NR; ++r) {
        const int x = first + row8 + r * 8;
        float q[D / 64][2][8];
        float top = 0.f;
        w.new_row[r] = x < u.n_rows ? x / p.group : -1;
        const int64_t at = int64_t(u.rr.r0 + x / p.group) * p.a.q_row_stride +
                           int64_t(u.head * p.group + x % p.group) * p.a.q_head_stride + t * 16;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                if (w.new_row[r] >= 0) {
                    load_q8(p.a.q, p.a.type, p.vec_q != 0, at + c * 64 + hf * 8, q[c][hf]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[c][hf][i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[c][hf][i]));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float to;
        query_factors(top, p.a.scale, to, w.rf[r]);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float *x4 = &q[c][j / 2][(j & 1) * 4];
                float2 a = make_float2(x4[0] * to, x4[1] * to), b = make_float2(x4[2] * to, x4[3] * to);
                if constexpr (MODE == kSplit) {
                    w.q[c * 4 + j][0] = split2(a, &w.q[c * 4 + j][1]);
                    w.q[c * 4 + j][2] = split2(b, &w.q[c * 4 + j][3]);
                } else {
                    w.q[c * 4 + j][r] = pack2(a);
                    w.q[c * 4 + j][2 + r] = pack2(b);
                }
            }
        w.m[r] = -INFINITY, w.l[r] = 0.f, w.E[r] = 40.f;
    }
#pragma unroll
    for (int j = 0; j < w.NJ; ++j)
#pragma unroll
        for (int i = 0; i < 2 * w.NR; ++i) w.o[j][i] = 0.f;
}

// One tile for a warp's rows.  st: the stage; ok: bit i says that page i of the tile exists.  Ends with a
// converged warp that reads the stage no more.
template <int D, int FORMAT, int MODE>
__device__ __forceinline__ void tile_rows(const AttnKv8 &p, const Unit &u, uint8_t *st, int tile, uint32_t ok, Rows<D, MODE> &w) {
    constexpr int NR = Rows<D, MODE>::NR, NJ = Rows<D, MODE>::NJ, kBlock = 16 * D, kChunks = D / 64;
    const int lane = threadIdx.x & 31, row8 = lane >> 2, t = lane & 3;
    const float *sc = reinterpret_cast<const float *>(st + 4 * kBlock);  // [k, v][page][16]
    const int p0 = tile * kAk8Tile;
    // only tiles that reach into the new rows, or miss a page, have masks
    const bool whole = p0 + kAk8Tile <= u.span.ctx && ok == 3u;
    if (!whole) {  // V codes that no position fills become zeros: a weight of 0 has to stay 0
        if (p0 + lane >= u.span.total || !(ok >> (lane >> 4) & 1u)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                *reinterpret_cast<uint4 *>(st + 2 * kBlock + lane * D + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
    }

    // scores, without the rows' factors; pair i = (page, tau) holds two neighbouring positions
    float2 sv[4][NR];
    {
        float c[4][4];  // four chains of products in turn: one alone waits for itself
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * (row8 >> 1) + 2 * (i & 1) + (row8 & 1);
                v[i] = *reinterpret_cast<const uint4 *>(st + (i >> 1) * kBlock + r * D + ch * 64 + t * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t(&qa)[4] = w.q[ch * 4 + j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t b0, b1;
                    codes_f16<FORMAT>(j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w, b0, b1);
                    if (ch == 0 && j == 0)
                        mma16816_0(c[i], qa[0], qa[1], qa[2], qa[3], b0, b1);
                    else
                        mma16816(c[i], qa[0], qa[1], qa[2], qa[3], b0, b1);
                }
            }
        }
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
            const float4 ks = *reinterpret_cast<const float4 *>(sc + pg * 16 + 4 * t);
#pragma unroll
            for (int tau = 0; tau < 2; ++tau) {
                const float2 k2 = tau ? make_float2(ks.z, ks.w) : make_float2(ks.x, ks.y);
                const float(&ci)[4] = c[pg * 2 + tau];
                if constexpr (MODE == kSplit) {
                    sv[pg * 2 + tau][0] = mul2(add2(make_float2(ci[0], ci[1]), make_float2(ci[2], ci[3])), k2);
                } else {
                    sv[pg * 2 + tau][0] = mul2(make_float2(ci[0], ci[1]), k2);
                    sv[pg * 2 + tau][1] = mul2(make_float2(ci[2], ci[3]), k2);
                }
            }
        }
    }
    uint32_t seen[NR];  // bit: page * 4 + position within the lane's four
    if (!whole) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            seen[r] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pos = p0 + (i >> 2) * kKv8Page + 4 * t + (i & 3), j = pos - u.span.ctx;
                bool in = pos < u.span.total && (ok >> (i >> 2) & 1u);
                if (in && j >= 0) {
                    if (w.new_row[r] < 0)
                        in = false;
                    else if (!p.a.mask)
                        in = j <= w.new_row[r];
                    else
                        in = j < 32 * p.a.mask_words &&
                             ((__ldg(p.a.mask + size_t(u.rr.r0 + w.new_row[r]) * p.a.mask_words + j / 32) >> (j & 31)) & 1u);
                }
                seen[r] |= in ? 1u << i : 0u;
                if (!in) ((i & 1) ? sv[i >> 1][r].y : sv[i >> 1][r].x) = -INFINITY;
            }
        }
    }
    // the running exponents of the V scales
    float E0[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) E0[r] = w.E[r];
    if (whole) {
        const float e = float(__reduce_max_sync(0xffffffffu, finite_bits(sc[32 + lane])) >> 23);
#pragma unroll
        for (int r = 0; r < NR; ++r) w.E[r] = fmaxf(w.E[r], e);
    } else {  // a row's are those that it sees
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (seen[r] >> i & 1u) b = max(b, finite_bits(sc[32 + (i >> 2) * kKv8Page + 4 * t + (i & 3)]));
            b = max(b, __shfl_xor_sync(0xffffffffu, b, 1));
            b = max(b, __shfl_xor_sync(0xffffffffu, b, 2));
            w.E[r] = fmaxf(w.E[r], float(b >> 23));
        }
    }
    float corr[NR];
    // softmax
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        float mx = fmaxf(fmaxf(fmaxf(sv[0][r].x, sv[0][r].y), fmaxf(sv[1][r].x, sv[1][r].y)),
                         fmaxf(fmaxf(sv[2][r].x, sv[2][r].y), fmaxf(sv[3][r].x, sv[3][r].y)));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m = fmaxf(w.m[r], mx), base = score_base(m), up = 140.f - w.E[r];
        corr[r] = sums_factor(w.m[r], m, w.rf[r], E0[r], w.E[r]);
        w.m[r] = m;
        const float2 base2 = make_float2(-base, -base), rf2 = make_float2(w.rf[r], w.rf[r]), up2 = make_float2(up, up);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 &x = sv[i][r];
            x = fma2(add2(x, base2), rf2, up2);
            x.x = ex2(x.x), x.y = ex2(x.y);
            sum = add2(sum, x);
        }
        w.l[r] = fmaf(w.l[r], corr[r], sum.x + sum.y);
    }
    // weights as the left operand
    uint32_t wa[2][4];  // [page]: tau 0 rows g, g + 8, tau 1 rows g, g + 8
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const float4 vs = *reinterpret_cast<const float4 *>(sc + 32 + pg * 16 + 4 * t);
#pragma unroll
        for (int tau = 0; tau < 2; ++tau) {
            const float2 v2 = tau ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y);
            float2 x[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                x[r] = mul2(sv[pg * 2 + tau][r], v2);
                if (!whole) {  // a masked position's scale may be anything, NaN included
                    if (!(seen[r] >> (pg * 4 + tau * 2) & 1u)) x[r].x = 0.f;
                    if (!(seen[r] >> (pg * 4 + tau * 2 + 1) & 1u)) x[r].y = 0.f;
                }
            }
            if constexpr (MODE == kSplit) {
                wa[pg][tau * 2] = split2(x[0], &wa[pg][tau * 2 + 1]);
            } else {
                wa[pg][tau * 2] = pack2(x[0]);
                wa[pg][tau * 2 + 1] = pack2(x[1]);
            }
        }
    }
    if constexpr (MODE != kSplit) {
        // most tiles raise no maximum
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[NR - 1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                w.o[j][0] *= corr[0], w.o[j][1] *= corr[0];
                w.o[j][2 * NR - 2] *= corr[NR - 1], w.o[j][2 * NR - 1] *= corr[NR - 1];
            }
        }
    }
    uint32_t vw[2][4][D / 32];  // [page][position][word]
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t *from = st + (2 + pg) * kBlock + (4 * t + i) * D + row8 * (D / 8);
            if constexpr (D == 64) {
                const uint2 v = *reinterpret_cast<const uint2 *>(from);
                vw[pg][i][0] = v.x, vw[pg][i][1] = v.y;
            } else {
                const uint4 v = *reinterpret_cast<const uint4 *>(from);
                vw[pg][i][0] = v.x, vw[pg][i][1] = v.y, vw[pg][i][2] = v.z, vw[pg][i][3] = v.w;
            }
        }
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t b0[2][2], b1[2][2];  // [page], of columns 4 k + 2 half and the next
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                codes_f16<FORMAT>(__byte_perm(vw[pg][0][k], vw[pg][1][k], half ? 0x7362 : 0x5140), b0[pg][0], b0[pg][1]);
                codes_f16<FORMAT>(__byte_perm(vw[pg][2][k], vw[pg][3][k], half ? 0x7362 : 0x5140), b1[pg][0], b1[pg][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float(&oj)[2 * NR] = w.o[4 * k + 2 * half + i];
                if constexpr (MODE == kSplit) {
                    float c[4];
                    mma16816_0(c, wa[0][0], wa[0][1], wa[0][2], wa[0][3], b0[0][i], b1[0][i]);
                    mma16816(c, wa[1][0], wa[1][1], wa[1][2], wa[1][3], b0[1][i], b1[1][i]);
                    const float2 y = fma2(make_float2(oj[0], oj[1]), make_float2(corr[0], corr[0]),
                                          add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])));
                    oj[0] = y.x, oj[1] = y.y;
                } else {
                    mma16816(oj, wa[0][0], wa[0][1], wa[0][2], wa[0][3], b0[0][i], b1[0][i]);
                    mma16816(oj, wa[1][0], wa[1][1], wa[1][2], wa[1][3], b0[1][i], b1[1][i]);
                }
            }
        }
    }
    __syncwarp();
}

// A warp's rows (from `first` on) to the output where `part` is NULL, else as sums, reference and l to part[row].
// Lane (g, t) has of its rows the elements 2 NJ t .. in two runs of NJ.
template <int D, int MODE>
__device__ __forceinline__ void finish_rows(const AttnKv8 &p, const Unit &u, int first, float *part, Rows<D, MODE> &w) {
    constexpr int NJ = Rows<D, MODE>::NJ;
    const int lane = threadIdx.x & 31, row8 = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < w.NR; ++r) {
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 1);
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 2);
        if (w.new_row[r] < 0) continue;
        const int x = first + row8 + r * 8;
        if (!part) {
            const float f = w.l[r] == 0.f ? 0.f : 1.f / w.l[r];
            const int64_t at = int64_t(u.rr.r0 + w.new_row[r]) * p.a.out_row_stride +
                               int64_t(u.head * p.group + x % p.group) * p.a.out_head_stride + t * (2 * NJ);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < NJ; j += 8) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = w.o[j + i][2 * r + e] * f;
                    store_out8(p.a.out, p.a.type, p.vec_out != 0, at + e * NJ + j, y);
                }
        } else {
            float *to = part + (row8 + r * 8) * (D + 4);
            const float f = part_factor(w.E[r], 140);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < NJ; j += 4)
                    *reinterpret_cast<float4 *>(to + t * (2 * NJ) + e * NJ + j) = make_float4(
                        w.o[j][2 * r + e] * f, w.o[j + 1][2 * r + e] * f, w.o[j + 2][2 * r + e] * f, w.o[j + 3][2 * r + e] * f);
            if (t == 0) to[D] = part_reference(w.m[r], w.rf[r]), to[D + 1] = w.l[r] * f;
        }
    }
}

// Units of the rows that one warp takes.
template <int D, int FORMAT, int MODE, bool DIRECT>
__global__ void __launch_bounds__(Ak8Shape<D>::kWarps * 32, 1) k_attn_kv8(const __grid_constant__ AttnKv8 p) {
    using S = Ak8Shape<D>;
    using W = Rows<D, MODE>;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t *plan = reinterpret_cast<uint32_t *>(smem + S::kRing);  // [n_seqs + 1]
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Run run{};
    run.g_end = 1;
    if (!DIRECT) {
        const int64_t total = plan_tiles<W::kRows, kAk8Tile, S::kWarps>(p, plan);
        if (!warp_run<S::kWarps>(p, total, run)) return;
    }
    uint8_t *ring = smem + warp * (S::kStage * S::kStages);
    const uint32_t ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

    while (run.g < run.g_end) {
        int status = 0;
        const Unit u = DIRECT ? direct_unit<W::kRows>(p, blockIdx.x, kAk8Tile, &status) : find_unit(p, plan, run, kAk8Tile);
        if (DIRECT && u.n_rows == 0) return;  // the whole CTA
        const int t1 = u.t1, t0 = u.t0 + (DIRECT ? warp : 0), step = DIRECT ? S::kWarps : 1;  // this warp's tiles

        // ---- the copies of a tile: lane i has the id of page i & 1, loaded a tile ahead of its use
        const auto page_id = [&](int tile) {
            const int i = 2 * tile + (lane & 1);
            return tile < t1 && i < u.n_pages ? kv8_page(p.cache, __ldg(u.table + i), &status) : -1;
        };
        const auto issue = [&](int stage, int id) { copy_pages<D, 2>(p.cache, u.head, ring_s + stage * S::kStage, id); };
        int ids[S::kStages];
#pragma unroll
        for (int i = 0; i < S::kStages; ++i) ids[i] = page_id(t0 + i * step);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            if (t0 + i * step < t1) issue(i, ids[i]);
            cp_async_commit();
        }
        W w;
        load_rows<D, MODE>(p, u, u.block * W::kRows, w);
        int stage = 0;
        for (int tile = t0; tile < t1; tile += step) {
            const uint32_t ok = __ballot_sync(0xffffffffu, ids[0] >= 0) & 3u;
            {
                int st = stage + S::kStages - 1;
                if (st >= S::kStages) st -= S::kStages;
                if (tile + (S::kStages - 1) * step < t1) issue(st, ids[S::kStages - 1]);
                cp_async_commit();
#pragma unroll
                for (int i = 0; i < S::kStages - 1; ++i) ids[i] = ids[i + 1];
                ids[S::kStages - 1] = page_id(tile + S::kStages * step);
            }
            cp_async_wait<S::kStages - 1>();
            __syncwarp();
            tile_rows<D, FORMAT, MODE>(p, u, ring + stage * S::kStage, tile, ok, w);
            if (++stage == S::kStages) stage = 0;
        }
        op_report(p.status, status);
        if (DIRECT) {
            finish_rows<D, MODE>(p, u, u.block * W::kRows, reinterpret_cast<float *>(ring), w);
            __syncthreads();
            join_warps<D, S::kWarps>(p, u, W::kRows, reinterpret_cast<const float *>(smem), S::kStage * S::kStages / 4);
            return;
        }
        finish_rows<D, MODE>(p, u, u.block * W::kRows,
                             u.t0 == 0 && t1 == u.tiles ? nullptr
                                                        : p.part + size_t(2 * run.item + (u.t0 == 0 ? 1 : 0)) * p.part_rows * (D + 4),
                             w);
        run.g += t1 - t0;
    }
}

// Units of more rows.  A CTA's four warps take 8 or 16 of them each; a tile is read once for all of
// them (64 rows of bf16 over an e4m3 cache of heads of 128: 171 TFLOP/s; three warps a scheduler wait for
// one another's shared-memory reads, 56% of that pipe, and products, 27% of theirs), and its codes are converted to fp16 once, each thread its share, a tile ahead of its use (the
// conversions are as many instructions as the rest of a tile's work).  The warps take their fragments
// from the converted tile with ldmatrix; its 16-byte chunks are stored at chunk ^ (row % 8).  A run
// belongs to a CTA.
template <int D>
struct Ak8Block {
    static constexpr int kWarps = 4, kCtas = 3, kStages = 4;  // CTAs of an SM
    static constexpr int kStage = 64 * D + 256;               // a tile as it is in the cache: 32 rows of K, of V, scales
    static constexpr int kTile = 128 * D;                     // the same in fp16
    static constexpr int kRing = kStage * kStages + 2 * kTile;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// A thread's share of a tile's codes, to fp16.  Positions that do not exist become zeros.
template <int D, int FORMAT>
__device__ __forceinline__ void convert_tile(const uint8_t *raw, uint8_t *to, int left, uint32_t ok) {
    constexpr uint32_t kGran = D / 16, kStep = 128 / kGran;  // 16-byte granules of a row of codes; rows between a thread's granules
    const uint32_t row = threadIdx.x / kGran, gr = threadIdx.x % kGran;  // row % 8 is the same in all of them
    raw += threadIdx.x * 16;
    uint8_t *to_a = to + row * (2 * D) + ((2 * gr) ^ (row & 7)) * 16, *to_b = to + row * (2 * D) + ((2 * gr + 1) ^ (row & 7)) * 16;
    uint4 w[64 / kStep];
#pragma unroll
    for (int i = 0; i < int(64 / kStep); ++i) w[i] = *reinterpret_cast<const uint4 *>(raw + i * 2048);
    if (left < kAk8Tile || ok != 3u) {
#pragma unroll
        for (int i = 0; i < int(64 / kStep); ++i) {
            const int pos = int(row + i * kStep) & 31;
            if (pos >= left || !(ok >> (pos >> 4) & 1u)) w[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
#pragma unroll
    for (int i = 0; i < int(64 / kStep); ++i) {
        uint4 a, b;
        codes_f16<FORMAT>(w[i].x, a.x, a.y);
        codes_f16<FORMAT>(w[i].y, a.z, a.w);
        codes_f16<FORMAT>(w[i].z, b.x, b.y);
        codes_f16<FORMAT>(w[i].w, b.z, b.w);
        *reinterpret_cast<uint4 *>(to_a + i * (kStep * 2 * D)) = a;
        *reinterpret_cast<uint4 *>(to_b + i * (kStep * 2 * D)) = b;
    }
}

template <int D, int FORMAT, int MODE>
__global__ void __launch_bounds__(128, Ak8Block<D>::kCtas) k_attn_kv8_block(const __grid_constant__ AttnKv8 p) {
    using S = Ak8Block<D>;
    constexpr int NR = MODE == kSplit ? 1 : 2, kWarpRows = 8 * NR, kRows = S::kWarps * kWarpRows, kBlock = 16 * D;
    constexpr int kBias = MODE == kHalf ? 134 : 140;  // of the weights' exponents
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t *plan = reinterpret_cast<uint32_t *>(smem + S::kRing);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row8 = lane >> 2, t = lane & 3, H = p.cache.kv_heads;
    const int64_t total = plan_tiles<kRows, kAk8Tile, S::kWarps>(p, plan);
    const int used = runs_used(total, p.runs);
    const uint32_t ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), half_s = ring_s + S::kStage * S::kStages;
    const uint32_t page_bytes = uint32_t(2 * kBlock) * uint32_t(H);

    for (int item = blockIdx.x; item < used * H; item += gridDim.x) {
        Run run;
        run.item = item;
        run.head = item % H;
        run.g = run_begin(total, used, item / H);
        run.g_end = run_begin(total, used, item / H + 1);
        while (run.g < run.g_end) {
            int status = 0;
            const Unit u = find_unit(p, plan, run, kAk8Tile);
            const int t0 = u.t0, t1 = u.t1;
            const auto page_id = [&](int tile) {
                const int i = 2 * tile + (lane & 1);
                return tile < t1 && i < u.n_pages ? kv8_page(p.cache, __ldg(u.table + i), &status) : -1;
            };
            // warp i copies page i & 1's K (i < 2) or V, and its scales (lanes 0 to 3)
            const uint8_t *codes = static_cast<const uint8_t *>(p.cache.codes) + ((warp >= 2 ? page_bytes / 2 : 0u) + u.head * kBlock + lane * 16);
            const float *scales = p.cache.scales + ((warp >= 2 ? H : 0) + u.head) * kKv8Page + (lane & 3) * 4;
            const uint32_t codes_to = ring_s + warp * kBlock + lane * 16, scales_to = ring_s + 4 * kBlock + warp * 64 + lane * 16;
            const auto issue = [&](int stage, int id) {
                const int page = __shfl_sync(0xffffffffu, id, warp & 1);
                if (page >= 0) {
                    const uint8_t *from = codes + uint64_t(uint32_t(page)) * page_bytes;
#pragma unroll
                    for (int i = 0; i < kBlock / 512; ++i) cp_async16(codes_to + stage * S::kStage + i * 512, from + i * 512);
                    if (lane < 4) cp_async16(scales_to + stage * S::kStage, scales + uint64_t(uint32_t(page)) * uint32_t(2 * kKv8Page * H));
                }
                cp_async_commit();
            };
            const auto pages_ok = [&](int id) { return __ballot_sync(0xffffffffu, id >= 0) & 3u; };
            int ids[S::kStages];  // of tiles t, t + 1, ..
#pragma unroll
            for (int i = 0; i < S::kStages; ++i) ids[i] = page_id(t0 + i);
#pragma unroll
            for (int i = 0; i < S::kStages - 1; ++i) issue(i, ids[i]);

            // ---- the query rows as fragments; the sign of the scale goes into them
            const int first = u.block * kRows + warp * kWarpRows;
            const bool any = first < u.n_rows;  // else the warp only copies and converts
            uint32_t q[D / 16][4];
            float rf[NR], m[NR], l[NR], E[NR], o[D / 8][2 * NR];
            int new_row[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int x = first + row8 + r * 8;
                new_row[r] = x < u.n_rows ? x / p.group : -1;
                const int64_t at = int64_t(u.rr.r0 + x / p.group) * p.a.q_row_stride +
                                   int64_t(u.head * p.group + x % p.group) * p.a.q_head_stride + 2 * t;
                float2 v[D / 8];
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    v[i] = new_row[r] >= 0 ? load_q2(p.a.q, p.a.type, at + i * 8) : make_float2(0.f, 0.f);
                    top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float to;
                query_factors(top, p.a.scale, to, rf[r]);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const float2 y = make_float2(v[i].x * to, v[i].y * to);
                    if constexpr (MODE == kSplit)
                        q[i / 2][2 * (i & 1)] = split2(y, &q[i / 2][2 * (i & 1) + 1]);
                    else
                        q[i / 2][2 * (i & 1) + r] = pack2(y);
                }
                m[r] = -INFINITY, l[r] = 0.f, E[r] = 40.f;
            }
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
#pragma unroll
                for (int i = 0; i < 2 * NR; ++i) o[j][i] = 0.f;

            cp_async_wait<S::kStages - 2>();
            __syncthreads();
            convert_tile<D, FORMAT>(smem, smem + S::kStage * S::kStages, u.span.total - t0 * kAk8Tile, pages_ok(ids[0]));
            int stage = 0;
            for (int tile = t0; tile < t1; ++tile, stage = (stage + 1) % S::kStages) {
                const uint32_t ok = pages_ok(ids[0]);
                cp_async_wait<S::kStages - 3>();
                __syncthreads();  // tile is converted and tile + 1 has arrived for all; tile - 1 is read by none
                issue((stage + S::kStages - 1) % S::kStages, ids[S::kStages - 1]);
#pragma unroll
                for (int i = 0; i < S::kStages - 1; ++i) ids[i] = ids[i + 1];
                ids[S::kStages - 1] = page_id(tile + S::kStages);
                if (tile + 1 < t1)
                    convert_tile<D, FORMAT>(smem + ((stage + 1) % S::kStages) * S::kStage,
                                            smem + S::kStage * S::kStages + ((stage + 1) & 1) * S::kTile,
                                            u.span.total - (tile + 1) * kAk8Tile, pages_ok(ids[0]));
                if (!any) continue;
                const float *sc = reinterpret_cast<const float *>(smem + stage * S::kStage + 4 * kBlock);  // [k, v][32]
                const uint32_t tile_s = half_s + (stage & 1) * S::kTile;
                const int p0 = tile * kAk8Tile;
                const bool whole = p0 + kAk8Tile <= u.span.ctx && ok == 3u;

                // scores without the rows' factors: of positions 8 j + 2 t and the next
                float2 sv[4][NR];
                {
                    float c[4][4];  // four chains of products in turn: one alone waits for itself
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        uint32_t b[4][4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            ldmatrix4(b[j], tile_s + (8 * j + (lane & 7)) * (2 * D) + ((4 * k + (lane >> 3)) ^ (lane & 7)) * 16);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (k == 0)
                                mma16816_0(c[j], q[0][0], q[0][1], q[0][2], q[0][3], b[j][0], b[j][1]);
                            else
                                mma16816(c[j], q[2 * k][0], q[2 * k][1], q[2 * k][2], q[2 * k][3], b[j][0], b[j][1]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma16816(c[j], q[2 * k + 1][0], q[2 * k + 1][1], q[2 * k + 1][2], q[2 * k + 1][3], b[j][2], b[j][3]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 k2 = *reinterpret_cast<const float2 *>(sc + 8 * j + 2 * t);
                        if constexpr (MODE == kSplit) {
                            sv[j][0] = mul2(add2(make_float2(c[j][0], c[j][1]), make_float2(c[j][2], c[j][3])), k2);
                        } else {
                            sv[j][0] = mul2(make_float2(c[j][0], c[j][1]), k2);
                            sv[j][NR - 1] = mul2(make_float2(c[j][2], c[j][3]), k2);
                        }
                    }
                }
                uint32_t seen[NR];  // bit: 2 j + (0 or 1)
                if (!whole) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        seen[r] = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int pos = p0 + 8 * (i >> 1) + 2 * t + (i & 1), j = pos - u.span.ctx;
                            bool in = pos < u.span.total && (ok >> (i >> 2) & 1u);
                            if (in && j >= 0) {
                                if (new_row[r] < 0)
                                    in = false;
                                else if (!p.a.mask)
                                    in = j <= new_row[r];
                                else
                                    in = j < 32 * p.a.mask_words &&
                                         ((__ldg(p.a.mask + size_t(u.rr.r0 + new_row[r]) * p.a.mask_words + j / 32) >> (j & 31)) & 1u);
                            }
                            seen[r] |= in ? 1u << i : 0u;
                            if (!in) ((i & 1) ? sv[i >> 1][r].y : sv[i >> 1][r].x) = -INFINITY;
                        }
                    }
                }
                // the tile's largest V scale, as its exponent, and its largest score, of each row
                float e[NR], mx[NR];
                if (whole) {
                    e[0] = e[NR - 1] = float(__reduce_max_sync(0xffffffffu, finite_bits(sc[32 + lane])) >> 23);
                } else {  // a row's are those that it sees
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        uint32_t b = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (seen[r] >> i & 1u) b = max(b, finite_bits(sc[32 + 8 * (i >> 1) + 2 * t + (i & 1)]));
                        b = max(b, __shfl_xor_sync(0xffffffffu, b, 1));
                        b = max(b, __shfl_xor_sync(0xffffffffu, b, 2));
                        e[r] = float(b >> 23);
                    }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    mx[r] = fmaxf(fmaxf(fmaxf(sv[0][r].x, sv[0][r].y), fmaxf(sv[1][r].x, sv[1][r].y)),
                                  fmaxf(fmaxf(sv[2][r].x, sv[2][r].y), fmaxf(sv[3][r].x, sv[3][r].y)));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                }
                // What the weights are relative to.  kHalf: m follows the maximum only when that is 2^6 above it (weights
                // stay below 2^14), as the sums, which stay in the products' accumulators, have to be multiplied then;
                // most tiles move nothing.
                float corr[NR];
                const auto follow = [&](int r, float m1) {
                    const float E1 = fmaxf(E[r], e[r]);
                    corr[r] = sums_factor(m[r], m1, rf[r], E[r], E1);
                    m[r] = m1, E[r] = E1, l[r] *= corr[r];
                };
                if constexpr (MODE == kHalf) {
                    bool above[NR], moves = false;
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        above[r] = (mx[r] - m[r]) * rf[r] > 6.f;
                        moves = moves || above[r] || e[r] > E[r];
                    }
                    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                        for (int r = 0; r < NR; ++r) follow(r, above[r] ? mx[r] : m[r]);
#pragma unroll
                        for (int j = 0; j < D / 8; ++j) {
                            o[j][0] *= corr[0], o[j][1] *= corr[0];
                            o[j][2 * NR - 2] *= corr[NR - 1], o[j][2 * NR - 1] *= corr[NR - 1];
                        }
                    }
                } else {
                    follow(0, fmaxf(m[0], mx[0]));
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float base = score_base(m[r]), up = float(kBias) - E[r];
                    const float2 base2 = make_float2(-base, -base), rf2 = make_float2(rf[r], rf[r]), up2 = make_float2(up, up);
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float2 &x = sv[j][r];
                        x = fma2(add2(x, base2), rf2, up2);
                        x.x = ex2(x.x), x.y = ex2(x.y);
                        sum = add2(sum, x);
                    }
                    l[r] += sum.x + sum.y;
                }
                uint32_t wa[2][4];  // the weights as the left operand, 16 positions each
                const auto weights = [&](auto masked) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v2 = *reinterpret_cast<const float2 *>(sc + 32 + 8 * j + 2 * t);
                        float2 x[NR];
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            x[r] = mul2(sv[j][r], v2);
                            if constexpr (decltype(masked)::value) {  // a masked position's scale may be anything, NaN included
                                if (!(seen[r] >> (2 * j) & 1u)) x[r].x = 0.f;
                                if (!(seen[r] >> (2 * j + 1) & 1u)) x[r].y = 0.f;
                            }
                        }
                        if constexpr (MODE == kSplit) {
                            wa[j / 2][2 * (j & 1)] = split2(x[0], &wa[j / 2][2 * (j & 1) + 1]);
                        } else {
                            wa[j / 2][2 * (j & 1)] = pack2(x[0]);
                            wa[j / 2][2 * (j & 1) + 1] = pack2(x[NR - 1]);
                        }
                    }
                };
                if (whole) weights(std::false_type()); else weights(std::true_type());
                const uint32_t v_s = tile_s + (32 + (lane & 15)) * (2 * D);  // the lane's row of the first 16
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {  // 16 columns
                    uint32_t b[2][4];
                    ldmatrix4_t(b[0], v_s + ((2 * j + (lane >> 4)) ^ (lane & 7)) * 16);
                    ldmatrix4_t(b[1], v_s + 16 * (2 * D) + ((2 * j + (lane >> 4)) ^ (lane & 7)) * 16);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float(&oj)[2 * NR] = o[2 * j + k];
                        if constexpr (MODE == kSplit) {
                            float c[4];
                            mma16816_0(c, wa[0][0], wa[0][1], wa[0][2], wa[0][3], b[0][2 * k], b[0][2 * k + 1]);
                            mma16816(c, wa[1][0], wa[1][1], wa[1][2], wa[1][3], b[1][2 * k], b[1][2 * k + 1]);
                            const float2 y = fma2(make_float2(oj[0], oj[1]), make_float2(corr[0], corr[0]),
                                                  add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])));
                            oj[0] = y.x, oj[1] = y.y;
                        } else {
                            mma16816(oj, wa[0][0], wa[0][1], wa[0][2], wa[0][3], b[0][2 * k], b[0][2 * k + 1]);
                            mma16816(oj, wa[1][0], wa[1][1], wa[1][2], wa[1][3], b[1][2 * k], b[1][2 * k + 1]);
                        }
                    }
                }
            }
            cp_async_wait<0>();
            __syncthreads();
            op_report(p.status, status);

            // ---- results: lane (g, t) has the elements 8 j + 2 t and the next of its rows
            const bool all = u.t0 == 0 && t1 == u.tiles;
            float *part = p.part + (size_t(2 * run.item + (u.t0 == 0 ? 1 : 0)) * p.part_rows + warp * kWarpRows + row8) * (D + 4);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                if (new_row[r] < 0) continue;
                const int x = first + row8 + r * 8;
                if (all) {
                    const float f = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        const float y[2] = {o[j][2 * r], o[j][2 * r + 1]};
                        store_row<2>(p, u.rr.r0 + new_row[r], u.head * p.group + x % p.group, 8 * j + 2 * t, y, f);
                    }
                } else {
                    float *to = part + r * 8 * (D + 4);
                    const float f = part_factor(E[r], kBias);
#pragma unroll
                    for (int j = 0; j < D / 8; ++j)
                        *reinterpret_cast<float2 *>(to + 8 * j + 2 * t) = make_float2(o[j][2 * r] * f, o[j][2 * r + 1] * f);
                    if (t == 0) to[D] = part_reference(m[r], rf[r]), to[D + 1] = l[r] * f;
                }
            }
            run.g += t1 - t0;
        }
    }
}

// The same for up to 4 query rows a unit (one new token of up to 4 heads a kv head): the products
// are turned over, K and V^T on the left (16 positions, 16 columns of V) and the rows, split into
// upper and lower parts, as the 8 columns on the right.  That takes half the products of the form
// above and leaves lane (g, t) with row t's scores of positions g' and g' + 8, g' = (g >> 1) + 4 (g & 1),
// of a page, so that four rows' softmax occupies every lane; movmatrix turns the weights into the
// right operand of w V.
template <int D, int FORMAT, bool DIRECT>
__global__ void __launch_bounds__(Ak8Few<D>::kWarps * 32, 1) k_attn_kv8_few(const __grid_constant__ AttnKv8 p) {
    using S = Ak8Few<D>;
    constexpr int NP = S::kPages, kTile = NP * kKv8Page;
    constexpr int NO = D / 8;                  // output columns a lane holds
    constexpr int kChunks = D / 64;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t *plan = reinterpret_cast<uint32_t *>(smem + S::kRing);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Run run{};
    run.g_end = 1;
    if (!DIRECT) {
        const int64_t total = plan_tiles<4, kTile, S::kWarps>(p, plan);
        if (!warp_run<S::kWarps>(p, total, run)) return;
    }

    uint8_t *ring = smem + warp * (S::kStage * S::kStages);
    const int row8 = lane >> 2, t = lane & 3;
    const int mine = (row8 >> 1) + 4 * (row8 & 1);  // the lane's first position in a page; the second is 8 on
    const uint32_t ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

    while (run.g < run.g_end) {
        int status = 0;
        const Unit u = DIRECT ? direct_unit<4>(p, blockIdx.x, kTile, &status) : find_unit(p, plan, run, kTile);
        if (DIRECT && u.n_rows == 0) return;  // the whole CTA
        const int t1 = u.t1, t0 = u.t0 + (DIRECT ? warp : 0), step = DIRECT ? S::kWarps : 1;  // this warp's tiles

        // ---- the copies of a tile: lane i has the id of page i % NP, loaded a tile ahead of its use
        const auto page_id = [&](int tile) {
            const int i = NP * tile + (lane & (NP - 1));
            return tile < t1 && i < u.n_pages ? kv8_page(p.cache, __ldg(u.table + i), &status) : -1;
        };
        const auto issue = [&](int stage, int id) { copy_pages<D, NP>(p.cache, u.head, ring_s + stage * S::kStage, id); };
        int ids[S::kStages];
#pragma unroll
        for (int i = 0; i < S::kStages; ++i) ids[i] = page_id(t0 + i * step);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            if (t0 + i * step < t1) issue(i, ids[i]);
            cp_async_commit();
        }

        // ---- the query: column g of the right operand is row g >> 1, upper part for even g, lower for odd
        uint32_t qf[D / 16][2];
        float rf;               // of row t
        {
            const int x = u.block * 4 + (row8 >> 1);
            float q[kChunks][2][8];
            float top = 0.f;
            const int64_t at = int64_t(u.rr.r0 + x / p.group) * p.a.q_row_stride +
                               int64_t(u.head * p.group + x % p.group) * p.a.q_head_stride + t * 16;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    if (x < u.n_rows) {
                        load_q8(p.a.q, p.a.type, p.vec_q != 0, at + c * 64 + hf * 8, q[c][hf]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) q[c][hf][i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[c][hf][i]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float to;
            query_factors(top, p.a.scale, to, rf);
            rf = __shfl_sync(0xffffffffu, rf, t * 8);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float *x4 = &q[c][j / 2][(j & 1) * 4];
                    uint32_t low[2];
                    qf[c * 4 + j][0] = split2(make_float2(x4[0] * to, x4[1] * to), &low[0]);
                    qf[c * 4 + j][1] = split2(make_float2(x4[2] * to, x4[3] * to), &low[1]);
                    if (row8 & 1) qf[c * 4 + j][0] = low[0], qf[c * 4 + j][1] = low[1];
                }
        }
        const int x_row = u.block * 4 + t;
        const int new_row = x_row < u.n_rows ? x_row / p.group : -1;

        float o[NO], m = -INFINITY, l = 0.f, E = 40.f;
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j] = 0.f;

        int stage = 0;
        for (int tile = t0; tile < t1; tile += step) {
            const int id_now = ids[0];
            {
                int st = stage + S::kStages - 1;
                if (st >= S::kStages) st -= S::kStages;
                if (tile + (S::kStages - 1) * step < t1) issue(st, ids[S::kStages - 1]);
                cp_async_commit();
#pragma unroll
                for (int i = 0; i < S::kStages - 1; ++i) ids[i] = ids[i + 1];
                ids[S::kStages - 1] = page_id(tile + S::kStages * step);
            }
            cp_async_wait<S::kStages - 1>();
            __syncwarp();
            uint8_t *st = ring + stage * S::kStage;
            const float *sc = reinterpret_cast<const float *>(st + 2 * NP * S::kBlock);  // [k, v][page][16]
            const int p0 = tile * kTile;
            const uint32_t ok = __ballot_sync(0xffffffffu, id_now >= 0) & ((1u << NP) - 1);
            const bool whole = p0 + kTile <= u.span.ctx && ok == (1u << NP) - 1;
            if (!whole) {  // V codes that no position fills become zeros: a weight of 0 has to stay 0
#pragma unroll
                for (int k = 0; k < NP / 2; ++k) {
                    const int r = lane + 32 * k;
                    if (p0 + r >= u.span.total || !(ok >> (r >> 4) & 1u)) {
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
                            *reinterpret_cast<uint4 *>(st + NP * S::kBlock + r * D + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                __syncwarp();
            }

            // scores of row t, without its factor
            float2 sv[NP];
            {
                float c[NP][4];  // a chain of products a page, in turn
#pragma unroll
                for (int ch = 0; ch < kChunks; ++ch) {
                    uint4 w0[NP], w1[NP];
#pragma unroll
                    for (int pg = 0; pg < NP; ++pg) {
                        const uint8_t *from = st + pg * S::kBlock + mine * D + ch * 64 + t * 16;
                        w0[pg] = *reinterpret_cast<const uint4 *>(from), w1[pg] = *reinterpret_cast<const uint4 *>(from + 8 * D);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int pg = 0; pg < NP; ++pg) {
                            uint32_t a0, a1, a2, a3;
                            codes_f16<FORMAT>(j == 0 ? w0[pg].x : j == 1 ? w0[pg].y : j == 2 ? w0[pg].z : w0[pg].w, a0, a2);
                            codes_f16<FORMAT>(j == 0 ? w1[pg].x : j == 1 ? w1[pg].y : j == 2 ? w1[pg].z : w1[pg].w, a1, a3);
                            if (ch == 0 && j == 0)
                                mma16816_0(c[pg], a0, a1, a2, a3, qf[0][0], qf[0][1]);
                            else
                                mma16816(c[pg], a0, a1, a2, a3, qf[ch * 4 + j][0], qf[ch * 4 + j][1]);
                        }
                }
#pragma unroll
                for (int pg = 0; pg < NP; ++pg)
                    sv[pg] = mul2(make_float2(c[pg][0] + c[pg][1], c[pg][2] + c[pg][3]), make_float2(sc[pg * 16 + mine], sc[pg * 16 + mine + 8]));
            }
            uint32_t seen = 0;  // bit: 2 page + (0 or 1)
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 2 * NP; ++i) {
                    const int pos = p0 + (i >> 1) * kKv8Page + mine + 8 * (i & 1), j = pos - u.span.ctx;
                    bool in = pos < u.span.total && (ok >> (i >> 1) & 1u);
                    if (in && j >= 0) {
                        if (new_row < 0)
                            in = false;
                        else if (!p.a.mask)
                            in = j <= new_row;
                        else
                            in = j < 32 * p.a.mask_words &&
                                 ((__ldg(p.a.mask + size_t(u.rr.r0 + new_row) * p.a.mask_words + j / 32) >> (j & 31)) & 1u);
                    }
                    seen |= in ? 1u << i : 0u;
                    if (!in) ((i & 1) ? sv[i >> 1].y : sv[i >> 1].x) = -INFINITY;
                }
            }
            // the running exponent of the V scales, of row t
            const float E0 = E;
            {
                uint32_t b = 0;
                if (whole) {
#pragma unroll
                    for (int k = 0; k < NP / 2; ++k) b = max(b, finite_bits(sc[NP * 16 + lane + 32 * k]));
                    b = __reduce_max_sync(0xffffffffu, b);
                } else {  // of what it sees
#pragma unroll
                    for (int i = 0; i < 2 * NP; ++i)
                        if (seen >> i & 1u) b = max(b, finite_bits(sc[NP * 16 + (i >> 1) * kKv8Page + mine + 8 * (i & 1)]));
#pragma unroll
                    for (int i = 4; i < 32; i <<= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, i));
                }
                E = fmaxf(E, float(b >> 23));
            }
            // softmax over the lanes of equal t
            float mx = fmaxf(sv[0].x, sv[0].y);
#pragma unroll
            for (int i = 1; i < NP; ++i) mx = fmaxf(mx, fmaxf(sv[i].x, sv[i].y));
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
            const float m0 = m;
            m = fmaxf(m, mx);
            const float corr = sums_factor(m0, m, rf, E0, E), base = score_base(m), up = 140.f - E;
            const float2 base2 = make_float2(-base, -base), rf2 = make_float2(rf, rf), up2 = make_float2(up, up);
            float2 sum = make_float2(0.f, 0.f);
            uint32_t wb[NP][2];  // weights as the right operand
#pragma unroll
            for (int pg = 0; pg < NP; ++pg) {
                float2 x = fma2(add2(sv[pg], base2), rf2, up2);
                x.x = ex2(x.x), x.y = ex2(x.y);
                sum = add2(sum, x);
                float2 w = mul2(x, make_float2(sc[NP * 16 + pg * 16 + mine], sc[NP * 16 + pg * 16 + mine + 8]));
                if (!whole) {  // a masked position's scale may be anything, NaN included
                    if (!(seen >> (2 * pg) & 1u)) w.x = 0.f;
                    if (!(seen >> (2 * pg + 1) & 1u)) w.y = 0.f;
                }
                // (upper, lower) of each of the two positions, then row t to column 2 t and 2 t + 1
                const float2 up = __half22float2(__float22half2_rn(w));
                const uint32_t first = pack2(make_float2(up.x, w.x - up.x)), second = pack2(make_float2(up.y, w.y - up.y));
                asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(wb[pg][0]) : "r"(first));
                asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(wb[pg][1]) : "r"(second));
            }
            l = fmaf(l, corr, sum.x + sum.y);
            // w V: positions t, t + 4 (k = 2 t, 2 t + 1) and t + 8, t + 12 (k + 8) of a page
#pragma unroll
            for (int wp = 0; wp < D / 64; ++wp) {
                uint2 vw[NP][4];
#pragma unroll
                for (int pg = 0; pg < NP; ++pg)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vw[pg][i] = *reinterpret_cast<const uint2 *>(st + (NP + pg) * S::kBlock + (t + 4 * i) * D + row8 * (D / 8) + wp * 8);
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // columns 8 wp + 2 k, + 1 of the lane's
                    float c[4];
#pragma unroll
                    for (int pg = 0; pg < NP; ++pg) {
                        const uint32_t sel = k & 1 ? 0x7362 : 0x5140;
                        uint32_t a0, a1, a2, a3;
                        codes_f16<FORMAT>(__byte_perm(k < 2 ? vw[pg][0].x : vw[pg][0].y, k < 2 ? vw[pg][1].x : vw[pg][1].y, sel), a0, a1);
                        codes_f16<FORMAT>(__byte_perm(k < 2 ? vw[pg][2].x : vw[pg][2].y, k < 2 ? vw[pg][3].x : vw[pg][3].y, sel), a2, a3);
                        if (pg == 0)
                            mma16816_0(c, a0, a1, a2, a3, wb[0][0], wb[0][1]);
                        else
                            mma16816(c, a0, a1, a2, a3, wb[pg][0], wb[pg][1]);
                    }
                    o[wp * 8 + 2 * k] = fmaf(o[wp * 8 + 2 * k], corr, c[0] + c[1]);
                    o[wp * 8 + 2 * k + 1] = fmaf(o[wp * 8 + 2 * k + 1], corr, c[2] + c[3]);
                }
            }
            __syncwarp();  // the stage is free again
            if (++stage == S::kStages) stage = 0;
        }
        op_report(p.status, status);

        // ---- results: lane (g, t) has columns NO g .. of row t
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
        float *part = DIRECT ? reinterpret_cast<float *>(ring) : p.part + size_t(2 * run.item + (u.t0 == 0 ? 1 : 0)) * p.part_rows * (D + 4);
        if (DIRECT) __syncwarp();  // the ring is read no more
        if (new_row >= 0) {
            if (!DIRECT && u.t0 == 0 && t1 == u.tiles) {
                const float f = l == 0.f ? 0.f : 1.f / l;
                const int64_t at = int64_t(u.rr.r0 + new_row) * p.a.out_row_stride +
                                   int64_t(u.head * p.group + x_row % p.group) * p.a.out_head_stride + row8 * NO;
#pragma unroll
                for (int j = 0; j < NO; j += 8) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = o[j + i] * f;
                    store_out8(p.a.out, p.a.type, p.vec_out != 0, at + j, y);
                }
            } else {
                float *to = part + t * (D + 4);
                const float f = part_factor(E, 140);
#pragma unroll
                for (int j = 0; j < NO; j += 4)
                    *reinterpret_cast<float4 *>(to + row8 * NO + j) = make_float4(o[j] * f, o[j + 1] * f, o[j + 2] * f, o[j + 3] * f);
                if (row8 == 0) to[D] = part_reference(m, rf), to[D + 1] = l * f;
            }
        }
        if (DIRECT) {
            __syncthreads();
            join_warps<D, S::kWarps>(p, u, 4, reinterpret_cast<const float *>(smem), S::kStage * S::kStages / 4);
            return;
        }
        run.g += t1 - t0;
    }
}

// Merges the partial sums of units that were cut, in the order of their positions.  JOB_WARPS warps a
// (row, query head) take a share of its partials each, 32 at a time: the references first, one a lane, then
// the sums, whose loads then wait for nothing.
template <int D, int JOB_WARPS>
__global__ void __launch_bounds__(256) k_attn_kv8_join(const __grid_constant__ AttnKv8 p) {
    __shared__ float shares[JOB_WARPS > 1 ? JOB_WARPS : 1][D + 4];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t job = JOB_WARPS > 1 ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * 8 + warp;
    const int row = int(job / p.a.q_heads), qh = int(job - int64_t(row) * p.a.q_heads);
    if (row >= p.seqs.rows) return;
    RowOwner owner;
    if (!row_owner(p.seqs, row, row, row, owner)) return;
    const int s = owner.seq, H = p.cache.kv_heads, head = qh / p.group;
    const int x = (row - owner.r.r0) * p.group + (qh - head * p.group), block = x / p.tile_rows;
    const uint32_t before = __ldcg(p.plan + s), tiles = __ldcg(p.plan + p.seqs.n_seqs + 1 + s);
    const int64_t total = __ldcg(p.plan + p.seqs.n_seqs);
    if (total == 0) return;  // no plan
    const int used = runs_used(total, p.runs);
    const int64_t g0 = int64_t(before) + int64_t(block) * tiles, g1 = g0 + tiles;
    const int w0 = run_of(total, used, g0), w1 = run_of(total, used, g1 - 1);
    if (w0 == w1) return;  // written whole
    // run w0 begins the unit, the others begin inside it
    constexpr int E = D / 32;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    const size_t slot = size_t(p.part_rows) * (D + 4);
    const float *part = p.part + size_t(head) * 2 * slot + size_t(x - block * p.tile_rows) * (D + 4);
    const auto at = [&](int w) { return part + size_t(w) * H * 2 * slot + (w == w0 ? slot : 0); };
    const int share = JOB_WARPS > 1 ? (w1 - w0 + JOB_WARPS) / JOB_WARPS : w1 - w0 + 1;  // neighbouring partials of a warp
    const int first = JOB_WARPS > 1 ? w0 + warp * share : w0, last = JOB_WARPS > 1 ? min(w1, first + share - 1) : w1;
    for (int b = first; b <= last; b += 32) {
        const int n = min(32, last - b + 1);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < n) ml = __ldcg(reinterpret_cast<const float2 *>(at(b + lane) + D));
        float top = ml.x;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float m_new = fmaxf(m, top), ref = m_new == -INFINITY ? 0.f : m_new, old = ex2(m - ref), f = ex2(ml.x - ref);
        m = m_new;
        float sum = ml.y * f;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        l = fmaf(l, old, sum);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] *= old;
        for (int j0 = 0; j0 < n; j0 += 8) {
            float v[8][E];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float *from = at(b + min(j0 + j, n - 1));
                if constexpr (E == 2) {
                    const float2 y = __ldcg(reinterpret_cast<const float2 *>(from) + lane);
                    v[j][0] = y.x, v[j][1] = y.y;
                } else {
                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(from) + lane);
                    v[j][0] = y.x, v[j][1] = y.y, v[j][2] = y.z, v[j][3] = y.w;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float fj = __shfl_sync(0xffffffffu, f, j0 + j);
                if (j0 + j < n) {
#pragma unroll
                    for (int i = 0; i < E; ++i) o[i] = fmaf(v[j][i], fj, o[i]);
                }
            }
        }
    }
    if constexpr (JOB_WARPS > 1) {
#pragma unroll
        for (int i = 0; i < E; ++i) shares[warp][lane * E + i] = o[i];
        if (lane == 0) shares[warp][D] = m, shares[warp][D + 1] = l;
        __syncthreads();
        if (warp != 0) return;
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < JOB_WARPS; ++w) m = fmaxf(m, shares[w][D]);
        const float ref = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll
        for (int w = 0; w < JOB_WARPS; ++w) {
            const float f = ex2(shares[w][D] - ref);
            l = fmaf(shares[w][D + 1], f, l);
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = fmaf(shares[w][lane * E + i], f, o[i]);
        }
    }
    store_row<E>(p, row, qh, lane * E, o, l == 0.f ? 0.f : 1.f / l);
}

}  // namespace mossgpu
