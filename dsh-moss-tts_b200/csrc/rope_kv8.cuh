// rope_kv8.cuh -- rotary positions, quantising append and read-back of the 8-bit paged cache.
//
// All three are bound by HBM: an element is read once and written once, with a few instructions
// between.  Work goes to independent warps (no CTA barriers).  In k_rope_append LPH lanes (a power
// of two) share a head, 8 elements a lane, and a warp takes several heads of one row: a lane has the
// same columns in all of them, so its cosines and sines are computed once.
// Measured on one B200: rotation of 8191 rows of 40 heads of 128 (bf16, half layout) 36.9 us, 4.5 TB/s; append
// of 4232 rows of 32 + 8 + 8 such heads 30.7 us, 3.1 TB/s; read-back of 104,544 rows of 8 + 8 heads 117 us,
// 5.6 TB/s (stores of whole 32-byte sectors: 138 us with two 16-byte ones a lane).
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

// 32 bytes at once: a whole sector of a cache line from one lane.
__device__ __forceinline__ void load32(const void *p, uint4 &a, uint4 &b) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store32(void *p, const uint4 &a, const uint4 &b) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
                 "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
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

// A lane's share of a head is two chunks of 4 elements, at `first` and `second`.  kPairs: interleaved
// pairs (2i, 2i + 1) inside the chunks, which lie behind one another: one 16-byte vector in 16-bit types.
// kHalves: the half layout with a rotary_dim that is a multiple of 8; lane j < rotary_dim / 8 has elements
// 4j.. and their partners at rotary_dim / 2 + 4j.., the lanes behind it 8 neighbouring ones, so that no
// element has its partner in another lane.  Both move 8 to 32 bytes at a time.  kAny: either layout, any
// rotary_dim and alignment: element by element, partners by way of shared memory.
constexpr int kPairs = 0, kHalves = 1, kAny = 2;

// The two chunks of a lane, as they lie in memory.
template <typename T>
struct Raw8 {
    uint2 w[sizeof(T)];
};
template <typename T, int LAYOUT>
__device__ __forceinline__ Raw8<T> raw8(const T *p, int first, int second) {
    Raw8<T> r;
    if constexpr (LAYOUT == kAny) {
        T e[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = p[first + i], e[4 + i] = p[second + i];
        memcpy(&r, e, sizeof(r));
    } else if constexpr (sizeof(T) == 4 && LAYOUT == kPairs) {
        load32(p + first, reinterpret_cast<uint4 *>(&r)[0], reinterpret_cast<uint4 *>(&r)[1]);
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<uint4 *>(&r)[0] = *reinterpret_cast<const uint4 *>(p + first);
        reinterpret_cast<uint4 *>(&r)[1] = *reinterpret_cast<const uint4 *>(p + second);
    } else if constexpr (LAYOUT == kPairs) {
        *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(p + first);
    } else {
        r.w[0] = *reinterpret_cast<const uint2 *>(p + first);
        r.w[1] = *reinterpret_cast<const uint2 *>(p + second);
    }
    return r;
}
template <typename T, int LAYOUT>
__device__ __forceinline__ void put8(T *p, int first, int second, const float (&x)[8]) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = T(x[i]);
    Raw8<T> r;
    memcpy(&r, e, sizeof(r));
    if constexpr (LAYOUT == kAny) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[first + i] = e[i], p[second + i] = e[4 + i];
    } else if constexpr (sizeof(T) == 4 && LAYOUT == kPairs) {
        store32(p + first, reinterpret_cast<uint4 *>(&r)[0], reinterpret_cast<uint4 *>(&r)[1]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4 *>(p + first) = reinterpret_cast<uint4 *>(&r)[0];
        *reinterpret_cast<uint4 *>(p + second) = reinterpret_cast<uint4 *>(&r)[1];
    } else if constexpr (LAYOUT == kPairs) {
        *reinterpret_cast<uint4 *>(p + first) = *reinterpret_cast<uint4 *>(&r);
    } else {
        *reinterpret_cast<uint2 *>(p + first) = r.w[0];
        *reinterpret_cast<uint2 *>(p + second) = r.w[1];
    }
}
template <typename T>
__device__ __forceinline__ void raw_f32(const Raw8<T> &r, float (&x)[8]) {
    T e[8];
    memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = float(e[i]);
}

template <int LAYOUT>
struct LaneRope {
    float c[LAYOUT == kAny ? 8 : 4], s[LAYOUT == kAny ? 8 : 4];  // of pairs; kAny: of elements, the sine with its sign
    uint32_t mask;                                               // what turns
};
template <int LAYOUT>
__device__ __forceinline__ LaneRope<LAYOUT> lane_rope(const mossgpu_rope &r, int pos, int lane_in_head, bool inverse) {
    LaneRope<LAYOUT> t;
    t.mask = 0;
    if constexpr (LAYOUT == kAny) {
        const int half = r.rotary_dim / 2;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = lane_in_head * 8 + j;
            if (e < r.rotary_dim) {
                const bool first = r.interleaved ? !(e & 1) : e < half;
                const float2 v = rope_angle(pos, __ldg(r.steps + (r.interleaved ? e / 2 : first ? e : e - half)), r.magnitude, inverse);
                t.c[j] = v.x, t.s[j] = first ? -v.y : v.y;
                t.mask |= 1u << j;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = lane_in_head * 4 + k;  // the pair, in both layouts
            if (2 * i < r.rotary_dim) {
                const float2 v = rope_angle(pos, __ldg(r.steps + i), r.magnitude, inverse);
                t.c[k] = v.x, t.s[k] = v.y;
                t.mask |= 1u << k;
            }
        }
    }
    return t;
}
// x[0..3] and x[4..7]: the two chunks.  Elements that do not turn keep their values (the payload of a
// 16-bit NaN may change on its way through fp32).
// All lanes of the warp call the kAny form; `stage`: 256 floats of this warp, lph lanes a head.
template <int LAYOUT>
__device__ __forceinline__ void rope_turn(float (&x)[8], const LaneRope<LAYOUT> &t, const mossgpu_rope &r, float *stage, int lph) {
    if constexpr (LAYOUT == kAny) {
        const int lane = threadIdx.x & 31, half = r.rotary_dim / 2, base = (lane & (lph - 1)) * 8;
        const float *head = stage + (lane & ~(lph - 1)) * 8;
        __syncwarp();
        reinterpret_cast<float4 *>(stage + lane * 8)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(stage + lane * 8)[1] = make_float4(x[4], x[5], x[6], x[7]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = base + j;
            if (t.mask >> j & 1u) x[j] = x[j] * t.c[j] + head[r.interleaved ? e ^ 1 : e < half ? e + half : e - half] * t.s[j];
        }
    } else if (t.mask == 0xfu) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float &a = x[LAYOUT == kPairs ? 2 * k : k], &b = x[LAYOUT == kPairs ? 2 * k + 1 : k + 4];
            const float ya = a * t.c[k] - b * t.s[k];
            b = b * t.c[k] + a * t.s[k];
            a = ya;
        }
    } else if (t.mask) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float &a = x[LAYOUT == kPairs ? 2 * k : k], &b = x[LAYOUT == kPairs ? 2 * k + 1 : k + 4];
            if (t.mask >> k & 1u) {
                const float ya = a * t.c[k] - b * t.s[k];
                b = b * t.c[k] + a * t.s[k];
                a = ya;
            }
        }
    }
}

// One head of 8-bit codes: the scale from the absolute maximum over the group's lanes (compared as
// integers, which keeps NaN and infinity above every finite value), codes the nearest to the IEEE quotient
// x / scale, ties to even: a function of the values alone.  The quotient is first taken by the scale's
// approximate inverse, within 2^-22 of it; where the quotients 2^-20 below and above round to one code, so
// does what lies between.  Only a lane that this leaves open (about one in 500) divides.
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
    } else {
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
        const float inv_lo = inv * (1.f - 0x1p-20f), inv_hi = inv * (1.f + 0x1p-20f);
        if (format == MOSSGPU_KV_INT8) {
            constexpr float kRound = 12582912.f;  // 1.5 * 2^23: the sum's last bits are the nearest whole number
            uint32_t b[8];
            bool open = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                b[i] = __float_as_uint(fmaf(x[i], inv_lo, kRound));
                open |= b[i] != __float_as_uint(fmaf(x[i], inv_hi, kRound));
            }
            if (open) {
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = uint32_t(max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale)))));
            }
            c.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            c.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
        } else {
            uint32_t b[4];
            bool open = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * inv_lo, x[2 * i + 1] * inv_lo), __NV_SATFINITE, __NV_E4M3);
                open |= b[i] != __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * inv_hi, x[2 * i + 1] * inv_hi), __NV_SATFINITE, __NV_E4M3);
            }
            if (open) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    b[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale)), __NV_SATFINITE,
                                                    __NV_E4M3);
            }
            c.x = b[0] | b[1] << 16;
            c.y = b[2] | b[3] << 16;
        }
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
    int heads[2];            // of q, of k and v
    int rows, row_warps;     // warps that share a row
    int head_dim, inverse;
    int *status;
};

// The sequence that owns a row: its rows, slot and context.
struct RowOwner {
    RowRange r;
    int seq, slot, ctx;
};
// Of rows first .. last (the same in the whole warp), each lane's own `row`.  32 neighbouring sequences
// around where the rows would lie if all had as many are loaded at once, which finds them in one round
// trip in batches of up to 32 sequences and of equal ones; a search follows where it does not.
__device__ __forceinline__ bool row_owner(const mossgpu_seq_batch &q, int first, int last, int row, RowOwner &w) {
    const int lane = threadIdx.x & 31, n = q.n_seqs;
    const int b0 = n <= 32 ? 0 : max(0, min(n - 32, int(int64_t(first) * n / q.rows) - 8));
    const bool in = b0 + lane < n;
    int start = 0x7fffffff, end = 0x7fffffff, slot = -1, ctx = 0;
    if (in) {
        start = __ldg(q.row_start + b0 + lane), end = __ldg(q.row_start + b0 + lane + 1);
        slot = __ldg(q.slot + b0 + lane), ctx = __ldg(q.ctx_len + b0 + lane);
    }
    const bool covered = (b0 == 0 || __shfl_sync(0xffffffffu, start, 0) <= first) && (b0 + 32 >= n || last < __shfl_sync(0xffffffffu, end, 31));
    int s = -1;  // the last sequence that begins at or before the row
    if (covered) {
        if (first == last) {
            s = __popc(__ballot_sync(0xffffffffu, start <= row)) - 1;
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) s += __shfl_sync(0xffffffffu, start, j) <= row;
        }
        const int from = max(s, 0);
        if (s >= 0) s += b0;
        start = __shfl_sync(0xffffffffu, start, from), end = __shfl_sync(0xffffffffu, end, from);
        slot = __shfl_sync(0xffffffffu, slot, from), ctx = __shfl_sync(0xffffffffu, ctx, from);
    } else {
        s = warp_upper_bound(q.row_start, n, first) - 1;
        while (s + 1 < n && __ldg(q.row_start + s + 1) <= row) ++s;
        if (s >= 0) {
            start = __ldg(q.row_start + s), end = __ldg(q.row_start + s + 1);
            slot = __ldg(q.slot + s), ctx = __ldg(q.ctx_len + s);
        }
    }
    if (s < 0) return false;
    w.r = kv8_rows(start, end, q.rows);
    w.seq = s, w.slot = slot, w.ctx = ctx;
    return row >= w.r.r0 && row < w.r.r1;
}

// Where an owned row lies in the cache; page -1: nowhere (and *status says why).
struct RowPlace {
    int64_t at;   // position
    int page, off;
};
__device__ __forceinline__ RowPlace row_place(const mossgpu_kv8_cache &c, const RowOwner &o, int row, int *status) {
    const SeqSpan span = kv8_span(c, o.slot, o.ctx, o.r.r1 - o.r.r0, status);
    RowPlace w;
    w.at = int64_t(o.ctx) + (row - o.r.r0);
    w.page = -1, w.off = 0;
    if (w.at >= 0 && w.at < span.total) {
        w.off = int(w.at % kKv8Page);
        w.page = kv8_page(c, __ldg(c.page_table + size_t(o.slot) * c.pages_per_slot + w.at / kKv8Page), status);
    }
    return w;
}

// q (and, with KV, k) of a row turned, k and v quantised into the cache.  A pass is 32 / LPH heads of one
// tensor; the row's warps take the passes of q, k and v in turn.
template <typename T, int LPH, int LAYOUT, bool KV>
__global__ void __launch_bounds__(kRowThreads, KV ? 4 : 3) k_rope_append(const __grid_constant__ RowOp a) {
    constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;  // passes whose loads are in flight together
    constexpr int kHeads = 32 / LPH;                // heads a pass
    __shared__ __align__(16) float stage[LAYOUT == kAny ? kRowThreads * 8 : 4];
    const int lane = threadIdx.x & 31;
    const uint32_t job = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
    const uint32_t job_row = job / uint32_t(a.row_warps);
    if (job_row >= uint32_t(a.rows)) return;
    const int row = int(job_row), part = int(job - job_row * uint32_t(a.row_warps));
    const int in_head = lane & (LPH - 1), sub = lane / LPH, D = a.head_dim, rot = a.rope.rotary_dim;
    const bool here = in_head * 8 < D;
    int first = in_head * 8, second = first + 4;
    if (LAYOUT == kHalves && first < rot) first = in_head * 4, second = first + rot / 2;
    int pos = 0, page = -1, off = 0;
    if (KV) {
        RowOwner owner;
        if (!row_owner(a.seqs, row, row, row, owner)) return;  // the whole warp
        int status = 0;
        const RowPlace w = row_place(a.cache, owner, row, &status);
        if (lane == 0) op_report(a.status, status);
        pos = a.pos ? __ldg(a.pos + row) : int(w.at);
        page = w.page, off = w.off;
    } else {
        pos = __ldg(a.pos + row);
    }
    LaneRope<LAYOUT> turn;
    turn.mask = 0;
    if (rot > 0) turn = lane_rope<LAYOUT>(a.rope, pos, in_head, a.inverse != 0);
    float *st = LAYOUT == kAny ? stage + (threadIdx.x & ~31u) * 8 : stage;
    // the heads of one tensor, from this warp's first pass on; use(head, live, x) for each
    const auto run = [&](const void *src, int64_t row_stride, int64_t head_stride, int heads, int my_part, auto &&use) {
        const int step = a.row_warps * kHeads;
        const T *p = static_cast<const T *>(src) + row * row_stride + int64_t(my_part * kHeads + sub) * head_stride;
        for (int h0 = my_part * kHeads; h0 < heads; h0 += kAhead * step) {
            Raw8<T> raw[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (here && h0 + u * step + sub < heads) raw[u] = raw8<T, LAYOUT>(p, first, second);
                p += step * head_stride;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (h0 + u * step >= heads) break;  // the whole warp
                const int h = h0 + u * step + sub;
                const bool live = here && h < heads;
                float x[8];
                raw_f32(raw[u], x);
                use(h, live, x);
            }
        }
    };
    T *out_row = static_cast<T *>(a.q_out) + row * a.out_row_stride;
    run(a.src[0], a.row_stride[0], a.head_stride[0], a.heads[0], part, [&](int h, bool live, float (&x)[8]) {
        if (LAYOUT == kAny || live) rope_turn<LAYOUT>(x, turn, a.rope, st, LPH);
        if (live) put8<T, LAYOUT>(out_row + h * a.out_head_stride, first, second, x);
    });
    if constexpr (KV) {
        int before = (a.heads[0] + kHeads - 1) / kHeads;  // passes of the tensors before
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int my_part = (part + a.row_warps - before % a.row_warps) % a.row_warps;
            run(a.src[1 + half], a.row_stride[1 + half], a.head_stride[1 + half], a.heads[1], my_part, [&](int h, bool live, float (&x)[8]) {
                if (half == 0 && rot > 0 && (LAYOUT == kAny || live)) rope_turn<LAYOUT>(x, turn, a.rope, st, LPH);
                if (!live) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = 0.f;
                }
                float scale;
                const uint2 c = quantise8<LPH>(x, a.cache.format, &scale);
                if (live && page >= 0) {
                    const size_t cell = kv8_cell(a.cache, page, half, h, off);
                    uint8_t *codes = static_cast<uint8_t *>(a.cache.codes) + cell * size_t(LPH * 8);
                    if constexpr (LAYOUT == kHalves) {
                        *reinterpret_cast<uint32_t *>(codes + first) = c.x;
                        *reinterpret_cast<uint32_t *>(codes + second) = c.y;
                    } else {
                        *reinterpret_cast<uint2 *>(codes + first) = c;
                    }
                    if (in_head == 0) a.cache.scales[cell] = scale;
                }
            });
            before += (a.heads[1] + kHeads - 1) / kHeads;
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

// A warp takes kSets times kRows neighbouring rows, 16 codes a lane: positions of a page lie behind one
// another for each head, so that a load reads 512 contiguous bytes where the rows share a page.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) k_kv8_read(const __grid_constant__ ReadOp a) {
    constexpr int kLanes = D / 16, kRows = 32 / kLanes, kSets = 2, kAhead = 4;
    const int lane = threadIdx.x & 31;
    const uint32_t job = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5), group = job / uint32_t(a.row_warps);
    const int64_t from = int64_t(group) * (kRows * kSets);
    const int part = int(job - group * uint32_t(a.row_warps));
    if (from >= a.seqs.rows) return;
    const int row_z = int(min(from + kRows * kSets, int64_t(a.seqs.rows))) - 1;
    const int base = (lane & (kLanes - 1)) * 16, H = a.cache.kv_heads;
    int row[kSets];
    const uint8_t *codes[kSets];  // of the row's position in head 0 of K
    const float *scales[kSets];
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
        row[i] = int(min(from + i * kRows + lane / kLanes, int64_t(row_z)));  // lanes past the end repeat the last row
        RowOwner owner;
        const bool owned = row_owner(a.seqs, int(from), row_z, row[i], owner);
        RowPlace w{};
        int status = 0;
        if (owned) w = row_place(a.cache, owner, row[i], &status);
        op_report(a.status, status);
        codes[i] = nullptr;
        if (owned && w.page >= 0) {
            const size_t cell = kv8_cell(a.cache, w.page, 0, 0, w.off);
            codes[i] = static_cast<const uint8_t *>(a.cache.codes) + cell * D + base;
            scales[i] = a.cache.scales + cell;
        }
    }
    // item it < H: head it of K, else head it - H of V; they follow one another in the cache
    for (int it0 = part; it0 < 2 * H; it0 += kAhead * a.row_warps) {
        uint4 c[kAhead][kSets];
        float scale[kAhead][kSets];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int it = it0 + u * a.row_warps;
            if (it < 2 * H && a.out[it >= H]) {
#pragma unroll
                for (int i = 0; i < kSets; ++i)
                    if (codes[i]) {
                        c[u][i] = __ldg(reinterpret_cast<const uint4 *>(codes[i] + size_t(uint32_t(it) * uint32_t(kKv8Page * D))));
                        scale[u][i] = __ldg(scales[i] + it * kKv8Page);
                    }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int it = it0 + u * a.row_warps, half = it >= H;
            if (it < 2 * H && a.out[half]) {
                T *to = static_cast<T *>(a.out[half]) + (it - half * H) * a.head_stride[half] + base;
#pragma unroll
                for (int i = 0; i < kSets; ++i)
                    if (codes[i]) {
                        T *at = to + row[i] * a.row_stride[half];
                        float x[2][8];
                        dequantise8(c[u][i].x, c[u][i].y, a.cache.format, scale[u][i], x[0]);
                        dequantise8(c[u][i].z, c[u][i].w, a.cache.format, scale[u][i], x[1]);
                        if (a.vec[half]) {
                            T e[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) e[j] = T(x[j / 8][j % 8]);
                            uint4 w[sizeof(T)];
                            memcpy(w, e, sizeof(w));
#pragma unroll
                            for (int j = 0; j < int(sizeof(T)); j += 2) store32(reinterpret_cast<char *>(at) + j * 16, w[j], w[j + 1]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) at[j] = T(x[j / 8][j % 8]);
                        }
                    }
            }
        }
    }
}

}  // namespace mossgpu
