// rope_kv8.cuh -- rotary positions, quantising append and read-back of the 8-bit paged cache.
//
// One CTA per row.  LPH lanes (a power of two) share a head, 8 elements a lane; the CTA's groups
// take the row's heads in turn.  All three are bound by HBM: an element is read once and written
// once, and the arithmetic between is a few instructions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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

// Rotates the 8 elements base..base+7 of a head held by the lanes of a group; `stage` is this
// warp's 256 floats (the half layout fetches its partners from other lanes through it).  All
// lanes of the warp call it.
__device__ __forceinline__ void rope_turn(float (&x)[8], int base, int rot, bool inter, const float2 *tab, float *stage,
                                          int lph) {
    if (inter) {
#pragma unroll
        for (int m = 0; m < 4; ++m)
            if (base + 2 * m < rot) {
                const float2 t = tab[base / 2 + m];
                const float a = x[2 * m], b = x[2 * m + 1];
                x[2 * m] = a * t.x - b * t.y;
                x[2 * m + 1] = b * t.x + a * t.y;
            }
        return;
    }
    const int lane = threadIdx.x & 31, half = rot / 2;
    float *mine = stage + lane * 8, *head = stage + (lane & ~(lph - 1)) * 8;
    __syncwarp();
    reinterpret_cast<float4 *>(mine)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(mine)[1] = make_float4(x[4], x[5], x[6], x[7]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = base + j;
        if (e < rot) {
            const bool first = e < half;
            const float2 t = tab[first ? e : e - half];
            const float p = head[first ? e + half : e - half];
            x[j] = first ? x[j] * t.x - p * t.y : x[j] * t.x + p * t.y;
        }
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
    int head_dim, inverse;
    int *status;
};

// q (and k) of a row turned, k and v quantised into the cache.
template <typename T, int LPH>
__global__ void __launch_bounds__(kRowThreads) k_rope_append(const __grid_constant__ RowOp a) {
    __shared__ float2 tab[kMaxRopeDim / 2];
    __shared__ __align__(16) float stage[kRowThreads * 8];
    __shared__ int where[3];  // rotary position, page, offset in the page (-1: no such row or cell)
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    if (a.seqs.n_seqs > 0) {
        if (threadIdx.x < 32) {
            const int s = warp_upper_bound(a.seqs.row_start, a.seqs.n_seqs, row) - 1;
            int status = 0, pos = 0, page = -1, off = -1;
            if (s >= 0) {
                const RowRange r = kv8_rows(__ldg(a.seqs.row_start + s), __ldg(a.seqs.row_start + s + 1), a.seqs.rows);
                const int slot = __ldg(a.seqs.slot + s), ctx = __ldg(a.seqs.ctx_len + s);
                if (row >= r.r0 && row < r.r1) {
                    off = 0;
                    const SeqSpan span = kv8_span(a.cache, slot, ctx, r.r1 - r.r0, &status);
                    const int64_t at = int64_t(ctx) + (row - r.r0);
                    if (at >= 0 && at < span.total) {
                        off = int(at % kKv8Page);
                        page = kv8_page(a.cache, __ldg(a.cache.page_table + size_t(slot) * a.cache.pages_per_slot + at / kKv8Page),
                                        &status);
                    }
                    pos = a.pos ? __ldg(a.pos + row) : int(at);
                }
            }
            if (lane == 0) {
                where[0] = pos, where[1] = page, where[2] = off;
                op_report(a.status, status);
            }
        }
        __syncthreads();
        if (where[2] < 0) return;
    }
    const int rot = a.rope.rotary_dim;
    if (rot > 0) {
        const int pos = a.seqs.n_seqs > 0 ? where[0] : __ldg(a.pos + row);
        if (int(threadIdx.x) < rot / 2)
            tab[threadIdx.x] = rope_angle(pos, __ldg(a.rope.steps + threadIdx.x), a.rope.magnitude, a.inverse != 0);
        __syncthreads();
    }
    const int page = a.seqs.n_seqs > 0 ? where[1] : -1, off = a.seqs.n_seqs > 0 ? where[2] : 0;
    const int base = int(threadIdx.x % LPH) * 8, D = a.head_dim;
    float *st = stage + (threadIdx.x & ~31u) * 8;
    const int items = a.heads[0] + a.heads[1] + a.heads[2];
    constexpr int kGroups = kRowThreads / LPH;
    for (int it0 = 0; it0 < items; it0 += kGroups) {  // whole warps stay in the loop: rope_turn is warp-wide
        const int it = it0 + int(threadIdx.x) / LPH;
        const int kind = it < a.heads[0] ? 0 : it < a.heads[0] + a.heads[1] ? 1 : 2;
        const int h = kind == 0 ? it : kind == 1 ? it - a.heads[0] : it - a.heads[0] - a.heads[1];
        const bool live = it < items && base < D;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live)
            load8(static_cast<const T *>(a.src[kind]) + row * a.row_stride[kind] + h * a.head_stride[kind] + base,
                  a.vec[kind] != 0, x);
        if (rot > 0) {
            if (kind < 2 || !a.rope.interleaved) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = x[j];
                rope_turn(y, base, rot, a.rope.interleaved != 0, tab, st, LPH);
                if (kind < 2) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = y[j];
                }
            }
        }
        if (kind == 0) {
            if (live)
                store8(static_cast<T *>(a.q_out) + row * a.out_row_stride + h * a.out_head_stride + base, a.vec_out != 0, x);
        }
        if constexpr (LPH == 8 || LPH == 16) {  // head_dim 64, 128: the cache's
            if (__any_sync(0xffffffffu, kind > 0)) {
                float scale;
                const uint2 c = quantise8<LPH>(x, a.cache.format, &scale);
                if (live && kind > 0 && page >= 0) {
                    const size_t cell = kv8_cell(a.cache, page, kind - 1, h, off);
                    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.cache.codes) + cell * size_t(D) + base) = c;
                    if (base == 0) a.cache.scales[cell] = scale;
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
    int *status;
};

__device__ __forceinline__ float2 e4m3x2_f32(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3);
    return __half22float2(__half2(h));
}

template <typename T, int LPH>
__global__ void __launch_bounds__(kRowThreads) k_kv8_read(const __grid_constant__ ReadOp a) {
    __shared__ int where[2];
    const int row = blockIdx.x;
    if (threadIdx.x < 32) {
        const int s = warp_upper_bound(a.seqs.row_start, a.seqs.n_seqs, row) - 1;
        int status = 0, page = -1, off = 0;
        if (s >= 0) {
            const RowRange r = kv8_rows(__ldg(a.seqs.row_start + s), __ldg(a.seqs.row_start + s + 1), a.seqs.rows);
            const int slot = __ldg(a.seqs.slot + s), ctx = __ldg(a.seqs.ctx_len + s);
            if (row >= r.r0 && row < r.r1) {
                const SeqSpan span = kv8_span(a.cache, slot, ctx, r.r1 - r.r0, &status);
                const int64_t at = int64_t(ctx) + (row - r.r0);
                if (at >= 0 && at < span.total) {
                    off = int(at % kKv8Page);
                    page = kv8_page(a.cache, __ldg(a.cache.page_table + size_t(slot) * a.cache.pages_per_slot + at / kKv8Page),
                                    &status);
                }
            }
        }
        if (threadIdx.x == 0) {
            where[0] = page, where[1] = off;
            op_report(a.status, status);
        }
    }
    __syncthreads();
    const int page = where[0], off = where[1];
    if (page < 0) return;
    constexpr int D = LPH * 8;
    const int base = int(threadIdx.x % LPH) * 8;
    for (int it = int(threadIdx.x) / LPH; it < 2 * a.cache.kv_heads; it += kRowThreads / LPH) {
        const int half = it / a.cache.kv_heads, h = it - half * a.cache.kv_heads;
        if (!a.out[half]) continue;
        const size_t cell = kv8_cell(a.cache, page, half, h, off);
        const uint2 c = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.cache.codes) + cell * D + base));
        const float scale = __ldg(a.cache.scales + cell);
        float x[8];
        if (a.cache.format == MOSSGPU_KV_INT8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = float(int8_t(c.x >> (8 * i))) * scale;
                x[4 + i] = float(int8_t(c.y >> (8 * i))) * scale;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = e4m3x2_f32(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xffffu);
                x[2 * i] = f.x * scale;
                x[2 * i + 1] = f.y * scale;
            }
        }
        store8(static_cast<T *>(a.out[half]) + row * a.row_stride[half] + h * a.head_stride[half] + base, a.vec[half] != 0, x);
    }
}

}  // namespace mossgpu
