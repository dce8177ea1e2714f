// rope_kv8.cuh -- rotary positions, quantising append and read-back of the 8-bit paged cache.
//
// All three are bound by HBM: an element is read once and written once, with a few instructions
// between.  Work goes to independent warps (no CTA barriers).  In k_rope_append LPH lanes (a power
// of two) share a head, 8 elements a lane, and a warp takes several heads of one row: a lane has the
// same columns in all of them, so its cosines and sines are computed once.  The loads of kAhead
// passes are in flight together, the first of them issued before the row's place is looked up.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <string.h>

#include "kv8_index.h"

namespace mossgpu {

constexpr int kRowThreads = 256;
constexpr int kMaxRopeDim = 256;

__device__ __forceinline__ void op_report(int *status, int code) {
    if (code != 0 && status) atomicCAS(status, 0, code);
}

// 8 consecutive elements as fp32, 16 bytes at a time where `vec` says that this is aligned.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
            return;
        }
    } else {
        if (vec) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = float(e[i]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = float(p[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&x)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            uint4 a;
            T *e = reinterpret_cast<T *>(&a);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = T(x[i]);
            *reinterpret_cast<uint4 *>(p) = a;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = T(x[i]);
}

// Number of entries of the ascending a[0..n) that are <= v, by one warp: each step reads 32
// evenly spaced entries at once (two steps for a thousand sequences).
__device__ __forceinline__ int warp_upper_bound(const int32_t *a, int n, int v) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (len > 0) {
        const int step = (len + 31) / 32;
        const int at = lane * step;
        const bool le = at < len && __ldg(a + lo + at) <= v;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        if (c == 0) return lo;
        if (step == 1) return lo + c;
        lo += (c - 1) * step + 1;  // the probe itself is <= v
        len = min(step - 1, n - lo);
    }
    return lo;
}

// cos and sin of pos * step / 2^64 turns, times the magnitude.  The product wraps modulo a whole
// turn; its upper 32 bits as a signed fraction of half a turn leave an angle error below 2^-24.
__device__ __forceinline__ float2 rope_angle(int pos, uint64_t step, float magnitude, bool inverse) {
    const uint64_t phase = uint64_t(int64_t(pos)) * step;
    const float half_turns = float(int32_t(uint32_t(phase >> 32))) * 0x1p-31f;
    float s, c;
    sincospif(half_turns, &s, &c);
    return make_float2(c * magnitude, inverse ? -s * magnitude : s * magnitude);
}

// A lane's share of the rotation: elements base .. base + 7 of every head.  Interleaved, it holds
// both members of four pairs.  In the half layout the other member is rot / 2 elements away: in one
// other lane where rot is a multiple of 16 (shuffles), anywhere otherwise (through `stage`, 256
// floats of this warp).  The sine has its sign: y = x cos + partner sin.
struct LaneRope {
    float c[8], s[8];
    int turn;   // 0: nothing of this lane turns, 1: all, 2: some elements (mask)
    uint32_t mask;
};
__device__ __forceinline__ LaneRope lane_rope(const mossgpu_rope &r, int pos, int base, bool inverse) {
    LaneRope t;
    t.mask = 0;
    const int half = r.rotary_dim / 2;
    if (r.interleaved) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            t.c[2 * m] = t.c[2 * m + 1] = 1.f, t.s[2 * m] = t.s[2 * m + 1] = 0.f;
            if (base + 2 * m < r.rotary_dim) {
                const float2 v = rope_angle(pos, __ldg(r.steps + base / 2 + m), r.magnitude, inverse);
                t.c[2 * m] = t.c[2 * m + 1] = v.x;
                t.s[2 * m] = -v.y, t.s[2 * m + 1] = v.y;
                t.mask |= 3u << (2 * m);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = base + j;
            t.c[j] = 1.f, t.s[j] = 0.f;
            if (e < r.rotary_dim) {
                const bool first = e < half;
                const float2 v = rope_angle(pos, __ldg(r.steps + (first ? e : e - half)), r.magnitude, inverse);
                t.c[j] = v.x, t.s[j] = first ? -v.y : v.y;
                t.mask |= 1u << j;
            }
        }
    }
    t.turn = t.mask == 0 ? 0 : t.mask == 0xffu ? 1 : 2;
    return t;
}
// All lanes of the warp call it; `on`: this lane's head turns.
__device__ __forceinline__ void rope_turn(float (&x)[8], const mossgpu_rope &r, const LaneRope &t, bool on, int base, float *stage,
                                          int lph) {
    float p[8];
    if (r.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = x[j ^ 1];
    } else if (r.rotary_dim % 16 == 0) {
        const int lane = threadIdx.x & 31, d = r.rotary_dim / 16;
        const int from = t.turn ? (base < r.rotary_dim / 2 ? lane + d : lane - d) : lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = __shfl_sync(0xffffffffu, x[j], from);
    } else {
        const int lane = threadIdx.x & 31, half = r.rotary_dim / 2;
        const float *head = stage + (lane & ~(lph - 1)) * 8;
        __syncwarp();
        reinterpret_cast<float4 *>(stage + lane * 8)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(stage + lane * 8)[1] = make_float4(x[4], x[5], x[6], x[7]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = base + j;
            p[j] = e < r.rotary_dim ? head[e < half ? e + half : e - half] : 0.f;
        }
    }
    if (on && t.turn) {
        // elements past rotary_dim stay as they are, whatever their bits
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (t.turn == 1 || (t.mask >> j & 1u)) x[j] = x[j] * t.c[j] + p[j] * t.s[j];
    }
}

// One head of 8-bit codes: the scale from the absolute maximum over the group's lanes (compared
// as integers, which keeps NaN and infinity above every finite value), codes by an IEEE division
// and one rounding to nearest even, so that the codes are a function of the values alone.
template <int LPH>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], int format, float *scale_out) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool sound = top < 0x7f800000u;
    float scale = __fdiv_rn(__uint_as_float(top), format == MOSSGPU_KV_INT8 ? 127.f : 448.f);
    uint2 c = make_uint2(0u, 0u);
    if (!sound) {
        scale = __int_as_float(0x7fffffff);
    } else if (scale < 0x1p-126f) {
        scale = 0.f;
    } else if (format == MOSSGPU_KV_INT8) {
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = uint32_t(max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale))))) & 0xffu;
        c.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        c.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
    } else {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale)),
                                            __NV_SATFINITE, __NV_E4M3);
        c.x = b[0] | b[1] << 16;
        c.y = b[2] | b[3] << 16;
    }
    *scale_out = scale;
    return c;
}

struct RowOp {
    mossgpu_kv8_cache cache;
    mossgpu_seq_batch seqs;  // n_seqs 0: every row stands for itself (rotation alone)
    mossgpu_rope rope;       // rotary_dim 0: none
    const void *src[3];      // q, k, v
    void *q_out;             // may be src[0]
    int64_t row_stride[3], head_stride[3], out_row_stride, out_head_stride;
    const int32_t *pos;
    int heads[3];
    int vec[3], vec_out;
    int rows, row_warps;     // warps that share a row
    int head_dim, inverse;
    int *status;
};

// Where row `row` of a batch lies: its sequence s is at or after `first` (searched by the warp, or
// advanced by a lane).  Returns false where no sequence owns it.
struct RowPlace {
    int64_t at;   // position
    int page, off;
};
__device__ __forceinline__ bool row_place(const mossgpu_kv8_cache &c, const mossgpu_seq_batch &q, int s, int row, RowPlace &w,
                                          int *status) {
    if (s < 0) return false;
    const RowRange r = kv8_rows(__ldg(q.row_start + s), __ldg(q.row_start + s + 1), q.rows);
    const int slot = __ldg(q.slot + s), ctx = __ldg(q.ctx_len + s);
    if (row < r.r0 || row >= r.r1) return false;
    const SeqSpan span = kv8_span(c, slot, ctx, r.r1 - r.r0, status);
    w.at = int64_t(ctx) + (row - r.r0);
    w.page = -1, w.off = 0;
    if (w.at >= 0 && w.at < span.total) {
        w.off = int(w.at % kKv8Page);
        w.page = kv8_page(c, __ldg(c.page_table + size_t(slot) * c.pages_per_slot + w.at / kKv8Page), status);
    }
    return true;
}

template <typename T>
struct Raw8 {  // 8 elements as they lie in memory
    uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const T *p, bool vec) {
    Raw8<T> r;
    if (vec) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
        memcpy(&r, e, sizeof(r));
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void raw_f32(const Raw8<T> &r, float (&x)[8]) {
    T e[8];
    memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = float(e[i]);
}

// q (and k) of a row turned, k and v quantised into the cache.
template <typename T, int LPH>
__global__ void __launch_bounds__(kRowThreads) k_rope_append(const __grid_constant__ RowOp a) {
    constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;  // passes whose loads are in flight together
    constexpr int kHeads = 32 / LPH;                // heads a pass
    __shared__ __align__(16) float stage[kRowThreads * 8];
    const int lane = threadIdx.x & 31;
    const uint32_t job = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
    const uint32_t job_row = job / uint32_t(a.row_warps);
    if (job_row >= uint32_t(a.rows)) return;
    const int row = int(job_row), part = int(job - job_row * uint32_t(a.row_warps));
    const int base = (lane & (LPH - 1)) * 8, D = a.head_dim, hq = a.heads[0], hk = hq + a.heads[1], items = hk + a.heads[2];
    const auto head_of = [&](int it, int &kind) {
        kind = it < hq ? 0 : it < hk ? 1 : 2;
        return kind == 0 ? it : kind == 1 ? it - hq : it - hk;
    };
    const int step = a.row_warps * kHeads;  // this warp's passes: part * kHeads, + step, ...
    Raw8<T> raw[kAhead];
    const auto fetch = [&](int it0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int it = it0 + u * step + lane / LPH;
            int kind;
            const int h = head_of(it, kind);
            if (it < items && base < D)
                raw[u] = raw8(static_cast<const T *>(a.src[kind]) + row * a.row_stride[kind] + h * a.head_stride[kind] + base,
                              a.vec[kind] != 0);
        }
    };
    int it0 = part * kHeads;
    fetch(it0);
    int pos = 0, page = -1, off = 0;
    if (a.seqs.n_seqs > 0) {
        RowPlace w;
        int status = 0;
        const int s = warp_upper_bound(a.seqs.row_start, a.seqs.n_seqs, row) - 1;
        const bool owned = row_place(a.cache, a.seqs, s, row, w, &status);
        if (lane == 0) op_report(a.status, status);
        if (!owned) return;
        pos = a.pos ? __ldg(a.pos + row) : int(w.at);
        page = w.page, off = w.off;
    } else {
        pos = __ldg(a.pos + row);
    }
    LaneRope turn;
    const int rot = a.rope.rotary_dim;
    if (rot > 0) turn = lane_rope(a.rope, pos, base, a.inverse != 0);
    float *st = stage + (threadIdx.x & ~31u) * 8;
    for (; it0 < items; it0 += kAhead * step) {
        float x[kAhead][8];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw_f32(raw[u], x[u]);
        if (it0 + kAhead * step < items) fetch(it0 + kAhead * step);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (it0 + u * step >= items) break;  // the whole warp
            const int it = it0 + u * step + lane / LPH;
            int kind;
            const int h = head_of(it, kind);
            const bool live = it < items && base < D;
            if (!live) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[u][j] = 0.f;
            }
            if (rot > 0) rope_turn(x[u], a.rope, turn, kind < 2, base, st, LPH);
            if (kind == 0 && live)
                store8(static_cast<T *>(a.q_out) + row * a.out_row_stride + h * a.out_head_stride + base, a.vec_out != 0, x[u]);
            if constexpr (LPH == 8 || LPH == 16) {  // head_dim 64, 128: the cache's
                if (__any_sync(0xffffffffu, kind > 0 && live)) {
                    float scale;
                    const uint2 c = quantise8<LPH>(x[u], a.cache.format, &scale);
                    if (live && kind > 0 && page >= 0) {
                        const size_t cell = kv8_cell(a.cache, page, kind - 1, h, off);
                        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.cache.codes) + cell * size_t(D) + base) = c;
                        if (base == 0) a.cache.scales[cell] = scale;
                    }
                }
            }
        }
    }
}

struct ReadOp {
    mossgpu_kv8_cache cache;
    mossgpu_seq_batch seqs;
    void *out[2];
    int64_t row_stride[2], head_stride[2];
    int vec[2];
    int row_warps;
    int *status;
};

__device__ __forceinline__ float2 e4m3x2_f32(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3);
    return __half22float2(__half2(h));
}
// 8 codes as their values times the scale
__device__ __forceinline__ void dequantise8(uint32_t lo, uint32_t hi, int format, float scale, float (&x)[8]) {
    if (format == MOSSGPU_KV_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = float(int8_t(lo >> (8 * i))) * scale;
            x[4 + i] = float(int8_t(hi >> (8 * i))) * scale;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = e4m3x2_f32(((i < 2 ? lo : hi) >> (16 * (i & 1))) & 0xffffu);
            x[2 * i] = f.x * scale;
            x[2 * i + 1] = f.y * scale;
        }
    }
}

// A warp takes kRows neighbouring rows, 16 codes a lane: positions of a page lie behind one another
// for each head, so that a pass reads 512 contiguous bytes where the rows share a page.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) k_kv8_read(const __grid_constant__ ReadOp a) {
    constexpr int kLanes = D / 16, kRows = 32 / kLanes, kAhead = 4;
    const int lane = threadIdx.x & 31;
    const uint32_t job = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5), group = job / uint32_t(a.row_warps);
    const int64_t first = int64_t(group) * kRows;
    const int part = int(job - group * uint32_t(a.row_warps));
    if (first >= a.seqs.rows) return;
    const int row = int(min(first + lane / kLanes, int64_t(a.seqs.rows) - 1));  // lanes past the end repeat the last row
    int s = warp_upper_bound(a.seqs.row_start, a.seqs.n_seqs, int(first)) - 1;
    // further rows may belong to later sequences: the last one that begins at or before the row
    while (s + 1 < a.seqs.n_seqs && __ldg(a.seqs.row_start + s + 1) <= row) ++s;
    RowPlace w;
    int status = 0;
    const bool owned = row_place(a.cache, a.seqs, s, row, w, &status);
    op_report(a.status, status);
    const bool live = owned && w.page >= 0;
    const int base = (lane & (kLanes - 1)) * 16, H = a.cache.kv_heads;
    for (int it0 = part; it0 < 2 * H; it0 += kAhead * a.row_warps) {
        uint4 c[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int it = it0 + u * a.row_warps, half = it >= H;
            if (live && it < 2 * H && a.out[half]) {
                const size_t cell = kv8_cell(a.cache, w.page, half, it - half * H, w.off);
                c[u] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.cache.codes) + cell * D + base));
                scale[u] = __ldg(a.cache.scales + cell);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int it = it0 + u * a.row_warps, half = it >= H;
            if (live && it < 2 * H && a.out[half]) {
                T *to = static_cast<T *>(a.out[half]) + row * a.row_stride[half] + (it - half * H) * a.head_stride[half] + base;
                float x[8];
                dequantise8(c[u].x, c[u].y, a.cache.format, scale[u], x);
                store8(to, a.vec[half] != 0, x);
                dequantise8(c[u].z, c[u].w, a.cache.format, scale[u], x);
                store8(to + 8, a.vec[half] != 0, x);
            }
        }
    }
}

}  // namespace mossgpu
