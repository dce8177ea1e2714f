// attn_kv8.cuh -- attention of one or a few new rows a sequence over the 8-bit paged cache.
//
// Work.  A unit is (sequence, kv head, block of kTileRows query rows); its rows are the
// sequence's new rows times the query heads of the group, so a cache byte serves all of them.  A
// unit's positions come in tiles of 32 (two pages).  All tiles of all units, in order, are cut
// into equal runs, one per warp of the grid: however ragged the batch is, every warp has the same
// work.  A warp that has a whole unit writes its rows; a unit cut between warps leaves partial
// sums in the workspace, which k_attn_kv8_join (a dependent launch) merges in a fixed order, so
// that a result does not depend on timing.
//
// A tile.  The warp's own ring of tiles in shared memory is filled by cp.async (16 bytes a lane,
// no barrier but the warp's own).  S = q K^T and o += w V are mma.sync m16n8k16 products in fp16,
// in which every 8-bit code is exact.  Which element of the head dimension is the k-th of a
// product, and which position is the n-th, is free as long as both operands agree; here a lane
// takes 16 consecutive codes of a K row and, of four V rows, consecutive codes too, so that codes
// go from shared memory to a fragment by wide loads and conversions alone.  The scales of a
// position multiply its score (K) and its weight (V) in fp32.
//
// Precision.  A query row is scaled by a power of two to [128, 256) and rounded to fp16, exact for
// bf16 and fp16 inputs.  For bf16 outputs the weights w = p sv 2^(13 - E), E the exponent of the
// largest V scale so far, are rounded to fp16 as well (2^-11 against the output's 2^-8), 16 rows
// a product.  For fp32 and fp16 outputs both are split into an upper and a lower fp16 part (22
// bits) that occupy rows g and g + 8 of the same product, 8 rows a product; since the tensor
// cores truncate when they accumulate, such products start from zero and are added in fp32.
// Statistics, sums and partials are fp32.
#pragma once

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

struct AttnKv8 {
    mossgpu_kv8_cache cache;
    mossgpu_seq_batch seqs;
    mossgpu_attention_kv8_args a;
    int group;       // query heads per kv head
    int workers;     // warps of the grid
    int tile_rows;   // rows of a unit
    int part_rows;   // rows a partial keeps
    int vec_q, vec_out;
    uint32_t *plan;  // [n_seqs + 1] tiles (over row blocks, per kv head) before a sequence; then [n_seqs] tiles of one block
    float *part;     // [2 * workers][part_rows][head_dim + 4]: sums, then m (log2 units) and l
    int *status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ uint32_t pack2(float a, float b) { return half2_bits(__floats2half2_rn(a, b)); }
// the fp16 parts of (a, b): upper returned, lower = what the upper leaves
__device__ __forceinline__ uint32_t split2(float a, float b, uint32_t *lower) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *lower = pack2(a - f.x, b - f.y);
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

// 16-byte granule `gr` of row r (0..15) of a block, in the order that makes the K and the V reads
// of a tile free of bank conflicts.
template <int D>
__device__ __forceinline__ int granule(int r, int gr) {
    const int x = D == 64 ? (r & 2) : (((r & 1) << 2) | (r & 2));
    return r * (D / 16) + (gr ^ x);
}

// Position, within a page, of the n-th column of the tau-th product (n = 2 t + e).
__device__ __forceinline__ int page_row(int tau, int t, int e) { return ((t + e) & 3) + 4 * (2 * tau + e); }

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
__device__ __forceinline__ void store_out8(void *o, int type, bool vec, int64_t at, const float (&x)[8]) {
    if (type == MOSSGPU_F32)
        store8(static_cast<float *>(o) + at, vec, x);
    else if (type == MOSSGPU_F16)
        store8(static_cast<__half *>(o) + at, vec, x);
    else
        store8(static_cast<__nv_bfloat16 *>(o) + at, vec, x);
}

// Worker w has the tiles [total w / n, total (w + 1) / n); n <= total.
__device__ __forceinline__ int64_t run_begin(int64_t total, int n, int w) { return total * w / n; }
__device__ __forceinline__ int run_of(int64_t total, int n, int64_t g) { return int(((g + 1) * n - 1) / total); }
__device__ __forceinline__ int runs_used(int64_t total, int workers) { return int(total < workers ? total : workers); }

template <int D, int FORMAT, bool SPLIT>
__global__ void __launch_bounds__(Ak8Shape<D>::kWarps * 32, 1) k_attn_kv8(const __grid_constant__ AttnKv8 p) {
    using S = Ak8Shape<D>;
    constexpr int kRows = SPLIT ? 8 : 16;      // rows of a unit
    constexpr int NR = SPLIT ? 1 : 2;          // rows a lane holds
    constexpr int NJ = D / 8;                  // output columns a lane holds, per row: 2 NJ
    constexpr int kGran = D / 16;              // granules of a row
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t *plan = reinterpret_cast<uint32_t *>(smem + S::kRing);  // [n_seqs + 1]
    __shared__ uint32_t warp_sum[S::kWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n_seqs = p.seqs.n_seqs, H = p.cache.kv_heads;

    // ---- tiles before each sequence
    {
        uint32_t before = 0;
        for (int s0 = 0; s0 < n_seqs; s0 += S::kWarps * 32) {
            const int s = s0 + int(threadIdx.x);
            uint32_t mine = 0;
            if (s < n_seqs) {
                const RowRange r = kv8_rows(__ldg(p.seqs.row_start + s), __ldg(p.seqs.row_start + s + 1), p.seqs.rows);
                int status = 0;
                if (r.r1 > r.r0) {
                    const SeqSpan span = kv8_span(p.cache, __ldg(p.seqs.slot + s), __ldg(p.seqs.ctx_len + s), r.r1 - r.r0, &status);
                    const uint32_t tiles = span.total > 0 ? (span.total + kAk8Tile - 1) / kAk8Tile : 1;
                    mine = tiles * uint32_t(((r.r1 - r.r0) * p.group + kRows - 1) / kRows);
                    if (blockIdx.x == 0) p.plan[n_seqs + 1 + s] = tiles;
                }
                if (blockIdx.x == 0) op_report(p.status, status);
            }
            uint32_t sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (lane == 31) warp_sum[warp] = sum;
            __syncthreads();
            uint32_t base = before, all = 0;
            for (int w = 0; w < S::kWarps; ++w) {
                if (w < warp) base += warp_sum[w];
                all += warp_sum[w];
            }
            if (s < n_seqs) plan[s] = base + sum - mine;
            before += all;
            __syncthreads();
        }
        if (threadIdx.x == 0) plan[n_seqs] = before;
        __syncthreads();
        if (blockIdx.x == 0)
            for (int s = threadIdx.x; s <= n_seqs; s += S::kWarps * 32) p.plan[s] = plan[s];
    }
    const int64_t total = int64_t(plan[n_seqs]) * H;
    const int used = runs_used(total, p.workers);
    const int worker = warp * gridDim.x + blockIdx.x;
    if (worker >= used) return;
    int64_t g = run_begin(total, used, worker);
    const int64_t g_end = run_begin(total, used, worker + 1);

    uint8_t *ring = smem + warp * (S::kStage * S::kStages);
    const uint32_t ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    const int row8 = lane >> 2, t = lane & 3;  // the lane's row and column pair in a product

    while (g < g_end) {
        // ---- which unit
        int lo = 0, hi = n_seqs;  // the last sequence that begins at or before g and has tiles
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (int64_t(plan[mid]) * H <= g) lo = mid; else hi = mid;
        }
        const int s = lo;
        const RowRange rr = kv8_rows(__ldg(p.seqs.row_start + s), __ldg(p.seqs.row_start + s + 1), p.seqs.rows);
        const int slot = __ldg(p.seqs.slot + s);
        int status = 0;
        const SeqSpan span = kv8_span(p.cache, slot, __ldg(p.seqs.ctx_len + s), rr.r1 - rr.r0, &status);
        status = 0;  // reported above
        const int tiles = span.total > 0 ? (span.total + kAk8Tile - 1) / kAk8Tile : 1;
        const int64_t rem = g - int64_t(plan[s]) * H;
        const int per_head = int(plan[s + 1] - plan[s]);
        const int head = int(rem / per_head);
        const int in_head = int(rem - int64_t(head) * per_head);
        const int block = in_head / tiles;
        const int t0 = in_head - block * tiles;
        const int t1 = int(min(int64_t(tiles), t0 + (g_end - g)));
        const int n_rows = (rr.r1 - rr.r0) * p.group;
        const int32_t *table = p.cache.page_table + size_t(span.total > 0 ? slot : 0) * p.cache.pages_per_slot;
        const int n_pages = (span.total + kKv8Page - 1) / kKv8Page;

        // ---- the copy of a tile into a stage; both pages' ids come one tile ahead
        const auto page_ids = [&](int tile) {
            int2 id = make_int2(-1, -1);
            if (2 * tile < n_pages) id.x = kv8_page(p.cache, __ldg(table + 2 * tile), &status);
            if (2 * tile + 1 < n_pages) id.y = kv8_page(p.cache, __ldg(table + 2 * tile + 1), &status);
            return id;
        };
        const auto issue = [&](int tile, int stage, int2 id) {
            const uint32_t dst = ring_s + uint32_t(stage * S::kStage);
            const uint8_t *codes = static_cast<const uint8_t *>(p.cache.codes);
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                const int page = pg ? id.y : id.x;
                const int left = page < 0 ? 0 : span.total - (2 * tile + pg) * kKv8Page;  // positions that exist
                const size_t k_cell = kv8_cell(p.cache, page < 0 ? 0 : page, 0, head, 0);
                const size_t v_cell = kv8_cell(p.cache, page < 0 ? 0 : page, 1, head, 0);
#pragma unroll
                for (int i = 0; i < kGran / 2; ++i) {
                    const int at = i * 32 + lane, r = at / kGran;
                    const uint32_t to = dst + uint32_t(pg * S::kBlock + granule<D>(r, at % kGran) * 16);
                    const int bytes = r < left ? 16 : 0;  // what no position fills becomes zeros
                    cp_async16(to, codes + k_cell * D + at * 16, bytes);
                    cp_async16(to + 2 * S::kBlock, codes + v_cell * D + at * 16, bytes);
                }
                if (lane < 8) {
                    const size_t cell = (lane < 4 ? k_cell : v_cell) + (lane & 3) * 4;
                    cp_async16(dst + uint32_t(4 * S::kBlock + ((lane >> 2) * 2 + pg) * 64 + (lane & 3) * 16), p.cache.scales + cell,
                               page < 0 ? 0 : 16);
                }
            }
            cp_async_commit();
        };

        int2 ids[S::kStages];
#pragma unroll
        for (int i = 0; i < S::kStages; ++i) ids[i] = t0 + i < t1 ? page_ids(t0 + i) : make_int2(-1, -1);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            if (t0 + i < t1) issue(t0 + i, i, ids[i]); else cp_async_commit();
        }

        // ---- the query rows as fragments
        uint32_t qf[D / 16][4];
        float rf[NR];           // what a product's value has to be multiplied by
        int new_row[NR];        // which new row of the sequence; -1: none
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int x = block * kRows + row8 + r * 8;
            float q[kGran / 4][2][8];
            float top = 0.f;
            new_row[r] = x < n_rows ? x / p.group : -1;
            const int64_t at = int64_t(rr.r0 + x / p.group) * p.a.q_row_stride +
                               int64_t(head * p.group + x % p.group) * p.a.q_head_stride + t * 16;
#pragma unroll
            for (int c = 0; c < kGran / 4; ++c)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    if (new_row[r] >= 0) {
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
            const int e = max(-110, min(110, int(__float_as_uint(top) >> 23) - 127));
            const float to = pow2i(7 - e);
            rf[r] = p.a.scale * 1.4426950408889634f * pow2i(e - 7);
#pragma unroll
            for (int c = 0; c < kGran / 4; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float *x4 = &q[c][j / 2][(j & 1) * 4];
                    if constexpr (SPLIT) {
                        qf[c * 4 + j][0] = split2(x4[0] * to, x4[1] * to, &qf[c * 4 + j][1]);
                        qf[c * 4 + j][2] = split2(x4[2] * to, x4[3] * to, &qf[c * 4 + j][3]);
                    } else {
                        qf[c * 4 + j][r] = pack2(x4[0] * to, x4[1] * to);
                        qf[c * 4 + j][2 + r] = pack2(x4[2] * to, x4[3] * to);
                    }
                }
        }

        float o[NJ][2 * NR], m[NR], l[NR];
        int E = 14;  // biased exponent of the largest V scale so far
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 2 * NR; ++i) o[j][i] = 0.f;
#pragma unroll
        for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.f;

        int2 id_now = ids[0], id_1 = ids[1], id_2 = S::kStages > 2 ? ids[S::kStages - 1] : make_int2(-1, -1);
        int stage = 0;
        for (int tile = t0; tile < t1; ++tile) {
            {
                const int ahead = tile + S::kStages - 1;
                const int2 id = S::kStages > 2 ? id_2 : id_1;
                int st = stage + S::kStages - 1;
                if (st >= S::kStages) st -= S::kStages;
                if (ahead < t1) issue(ahead, st, id); else cp_async_commit();
            }
            const int2 id_next = tile + S::kStages < t1 ? page_ids(tile + S::kStages) : make_int2(-1, -1);
            cp_async_wait<S::kStages - 1>();
            __syncwarp();
            const uint8_t *st = ring + stage * S::kStage;
            const float *sc = reinterpret_cast<const float *>(st + 4 * S::kBlock);  // [k, v][page][16]

            // scores
            float sv[2][2][2 * NR];  // [page][tau][row, e]
#pragma unroll
            for (int pg = 0; pg < 2; ++pg)
#pragma unroll
                for (int tau = 0; tau < 2; ++tau) {
                    const int r = page_row(tau, row8 >> 1, row8 & 1);
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ch = 0; ch < kGran / 4; ++ch) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(st + pg * S::kBlock + granule<D>(r, ch * 4 + t) * 16);
                        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t b0, b1;
                            codes_f16<FORMAT>(ww[j], b0, b1);
                            const uint32_t(&qa)[4] = qf[ch * 4 + j];
                            mma16816(c, qa[0], qa[1], qa[2], qa[3], b0, b1);
                        }
                    }
                    const float k0 = sc[pg * 16 + page_row(tau, t, 0)], k1 = sc[pg * 16 + page_row(tau, t, 1)];
                    if constexpr (SPLIT) {
                        sv[pg][tau][0] = (c[0] + c[2]) * (k0 * rf[0]);
                        sv[pg][tau][1] = (c[1] + c[3]) * (k1 * rf[0]);
                    } else {
                        sv[pg][tau][0] = c[0] * (k0 * rf[0]);
                        sv[pg][tau][1] = c[1] * (k1 * rf[0]);
                        sv[pg][tau][2] = c[2] * (k0 * rf[1]);
                        sv[pg][tau][3] = c[3] * (k1 * rf[1]);
                    }
                }
            // masks: only tiles that reach into the new rows, or miss a page, have any
            const int p0 = tile * kAk8Tile;
            const bool whole = p0 + kAk8Tile <= span.ctx && id_now.x >= 0 && id_now.y >= 0;
            uint32_t seen[NR];  // bit (pg * 4 + tau * 2 + e)
#pragma unroll
            for (int r = 0; r < NR; ++r) seen[r] = 0xffu;
            if (!whole) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    seen[r] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int pos = p0 + (i >> 2) * kKv8Page + page_row((i >> 1) & 1, t, i & 1);
                        bool ok = pos < span.total && ((i >> 2) ? id_now.y : id_now.x) >= 0;
                        const int j = pos - span.ctx;
                        if (ok && j >= 0) {
                            if (new_row[r] < 0)
                                ok = false;
                            else if (!p.a.mask)
                                ok = j <= new_row[r];
                            else
                                ok = j < 32 * p.a.mask_words &&
                                     ((__ldg(p.a.mask + size_t(rr.r0 + new_row[r]) * p.a.mask_words + j / 32) >> (j & 31)) & 1u);
                        }
                        seen[r] |= ok ? 1u << i : 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!(seen[r] >> i & 1u)) {
                            sv[i >> 2][(i >> 1) & 1][2 * r + (i & 1)] = -INFINITY;
                        }
                }
            }
            // the running exponent of the V scales
            int E_new;
            {
                const int pos = p0 + lane;
                uint32_t b = 0;
                if (pos < span.total) b = __float_as_uint(sc[32 + lane]) & 0x7fffffffu;
                if (b >= 0x7f800000u) b = 0;
                E_new = max(E, int(__reduce_max_sync(0xffffffffu, b) >> 23));
            }
            const float v_to = pow2i(140 - E_new), v_fix = E_new - E > 126 ? 0.f : pow2i(E - E_new);
            E = E_new;
            // softmax
            float corr[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sv[i >> 2][(i >> 1) & 1][2 * r + (i & 1)]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m_new = fmaxf(m[r], mx);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                corr[r] = exp2_approx(m[r] - ref);
                m[r] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float &x = sv[i >> 2][(i >> 1) & 1][2 * r + (i & 1)];
                    x = exp2_approx(x - ref);
                    sum += x;
                }
                l[r] = fmaf(l[r], corr[r], sum);
                corr[r] *= v_fix;
            }
            if constexpr (!SPLIT) {
                // the sums stay in the products' accumulators
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[j][0] *= corr[0], o[j][1] *= corr[0];
                    o[j][2] *= corr[1], o[j][3] *= corr[1];
                }
            }
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                uint32_t wa[4];  // the weights as the left operand: tau 0 rows g, g + 8, tau 1 rows g, g + 8
#pragma unroll
                for (int tau = 0; tau < 2; ++tau) {
                    const float v0 = sc[32 + pg * 16 + page_row(tau, t, 0)] * v_to, v1 = sc[32 + pg * 16 + page_row(tau, t, 1)] * v_to;
                    const int bit = pg * 4 + tau * 2;
                    // a masked position's scale may be anything, NaN included
                    const auto weight = [&](int r, int e, float v) {
                        return (seen[r] >> (bit + e) & 1u) ? sv[pg][tau][2 * r + e] * v : 0.f;
                    };
                    if constexpr (SPLIT) {
                        wa[tau * 2] = split2(weight(0, 0, v0), weight(0, 1, v1), &wa[tau * 2 + 1]);
                    } else {
                        wa[tau * 2] = pack2(weight(0, 0, v0), weight(0, 1, v1));
                        wa[tau * 2 + 1] = pack2(weight(1, 0, v0), weight(1, 1, v1));
                    }
                }
                uint32_t vw[4][D / 32];  // [2 tau + e][word]
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = page_row(i >> 1, t, i & 1);
                    const uint8_t *src = st + 2 * S::kBlock + pg * S::kBlock;
                    if constexpr (D == 64) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(src + granule<D>(r, row8 >> 1) * 16 + (row8 & 1) * 8);
                        vw[i][0] = w.x, vw[i][1] = w.y;
                    } else {
                        const uint4 w = *reinterpret_cast<const uint4 *>(src + granule<D>(r, row8) * 16);
                        vw[i][0] = w.x, vw[i][1] = w.y, vw[i][2] = w.z, vw[i][3] = w.w;
                    }
                }
#pragma unroll
                for (int w = 0; w < D / 32; ++w)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t b0[2], b1[2];  // of columns 4 w + 2 half and the next
                        codes_f16<FORMAT>(__byte_perm(vw[0][w], vw[1][w], half ? 0x7362 : 0x5140), b0[0], b0[1]);
                        codes_f16<FORMAT>(__byte_perm(vw[2][w], vw[3][w], half ? 0x7362 : 0x5140), b1[0], b1[1]);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float(&oj)[2 * NR] = o[4 * w + 2 * half + k];
                            if constexpr (SPLIT) {
                                float c[4] = {0.f, 0.f, 0.f, 0.f};
                                mma16816(c, wa[0], wa[1], wa[2], wa[3], b0[k], b1[k]);
                                oj[0] = (pg == 0 ? oj[0] * corr[0] : oj[0]) + (c[0] + c[2]);
                                oj[1] = (pg == 0 ? oj[1] * corr[0] : oj[1]) + (c[1] + c[3]);
                            } else {
                                mma16816(oj, wa[0], wa[1], wa[2], wa[3], b0[k], b1[k]);
                            }
                        }
                    }
            }
            __syncwarp();  // the stage is free again
            id_now = id_1;
            if constexpr (S::kStages > 2) {
                id_1 = id_2;
                id_2 = id_next;
            } else {
                id_1 = id_next;
            }
            if (++stage == S::kStages) stage = 0;
        }
        cp_async_wait<0>();
        __syncwarp();
        op_report(p.status, status);

        // ---- results: lane (g, t) has of its rows the elements 16 t NJ/8 .. in two runs of NJ
        const bool all = t0 == 0 && t1 == tiles;
        const float v_back = pow2i(max(-126, E - 140));
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (new_row[r] < 0) continue;
            const int x = block * kRows + row8 + r * 8;
            if (all) {
                const float f = l[r] == 0.f ? 0.f : v_back / l[r];
                const int64_t at = int64_t(rr.r0 + new_row[r]) * p.a.out_row_stride +
                                   int64_t(head * p.group + x % p.group) * p.a.out_head_stride + t * (2 * NJ);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < NJ; j += 8) {
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = o[j + i][2 * r + e] * f;
                        store_out8(p.a.out, p.a.type, p.vec_out != 0, at + e * NJ + j, y);
                    }
            } else {
                float *part = p.part + (size_t(2 * worker + (t0 == 0 ? 1 : 0)) * p.part_rows + (row8 + r * 8)) * (D + 4);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < NJ; j += 4)
                        *reinterpret_cast<float4 *>(part + t * (2 * NJ) + e * NJ + j) =
                            make_float4(o[j][2 * r + e] * v_back, o[j + 1][2 * r + e] * v_back, o[j + 2][2 * r + e] * v_back,
                                        o[j + 3][2 * r + e] * v_back);
                if (t == 0) part[D] = m[r], part[D + 1] = l[r];
            }
        }
        g += t1 - t0;
    }
}

// One warp per (row, query head): merges the partial sums of a unit that was cut, in the order of
// its positions.
template <int D>
__global__ void __launch_bounds__(256) k_attn_kv8_join(const __grid_constant__ AttnKv8 p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t job = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int row = int(job / p.a.q_heads), qh = int(job - int64_t(row) * p.a.q_heads);
    if (row >= p.seqs.rows) return;
    const int s = warp_upper_bound(p.seqs.row_start, p.seqs.n_seqs, row) - 1;
    if (s < 0) return;
    const RowRange rr = kv8_rows(__ldg(p.seqs.row_start + s), __ldg(p.seqs.row_start + s + 1), p.seqs.rows);
    if (row >= rr.r1) return;
    const int H = p.cache.kv_heads, head = qh / p.group;
    const int x = (row - rr.r0) * p.group + (qh - head * p.group), block = x / p.tile_rows;
    const uint32_t before = __ldcg(p.plan + s), after = __ldcg(p.plan + s + 1), tiles = __ldcg(p.plan + p.seqs.n_seqs + 1 + s);
    const int64_t total = int64_t(__ldcg(p.plan + p.seqs.n_seqs)) * H;
    const int used = runs_used(total, p.workers);
    const int64_t g0 = int64_t(before) * H + int64_t(head) * (after - before) + int64_t(block) * tiles, g1 = g0 + tiles;
    const int w0 = run_of(total, used, g0), w1 = run_of(total, used, g1 - 1);
    if (w0 == w1) return;  // written whole
    // worker w0 begins the unit at its run's second place unless the run itself begins here
    constexpr int E = D / 32;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    const size_t in_slot = size_t(x - block * p.tile_rows) * (D + 4);
    const size_t slot = size_t(p.part_rows) * (D + 4);
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) {
        const float *part = p.part + size_t(2 * w + (w == w0 ? 1 : 0)) * slot + in_slot;
        float v[E];
        if constexpr (E == 2) {
            const float2 a = __ldcg(reinterpret_cast<const float2 *>(part) + lane);
            v[0] = a.x, v[1] = a.y;
        } else {
            const float4 a = __ldcg(reinterpret_cast<const float4 *>(part) + lane);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        }
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part + D));
        const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
        const float fa = exp2_approx(m - ref), fb = exp2_approx(ml.x - ref);
        m = m_new;
        l = l * fa + ml.y * fb;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = o[i] * fa + v[i] * fb;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = int64_t(row) * p.a.out_row_stride + int64_t(qh) * p.a.out_head_stride + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = o[i] * f;
        if (p.a.type == MOSSGPU_F32)
            static_cast<float *>(p.a.out)[at + i] = y;
        else if (p.a.type == MOSSGPU_F16)
            static_cast<__half *>(p.a.out)[at + i] = __float2half_rn(y);
        else
            static_cast<__nv_bfloat16 *>(p.a.out)[at + i] = __float2bfloat16_rn(y);
    }
}

}  // namespace mossgpu
