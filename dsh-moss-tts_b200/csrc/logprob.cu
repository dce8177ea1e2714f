// logprob.cu -- log-probabilities of given tokens, entropy and the most likely tokens of rows of
// logits (mossgpu_token_logprobs).
//
// A row is held by one CTA or by a cluster of up to 16, 2 or 8 vectors of 16 bytes a thread in
// registers or 8 in registers and 8 in shared memory: it is read from HBM once, and the maximum, the
// sums and the selection all work on what was read.  With x the logits, M = max x, t = (x - M) log2(e) / T:
//   Z = sum 2^t,  S = sum 2^t t,
//   log p_i = (x_i - M) / T - ln Z,  entropy = ln Z - ln 2 S / Z.
// CTAs of a cluster sum against their own maxima; rank 0 merges.
//
// Selection: the threads form 32 groups; the k-th largest of the groups' maxima bounds the k-th
// largest logit from below, so only logits from it on are candidates: for k of 32 groups about
// -32 ln(1 - k / 32) are expected (9 for k = 8, 31 for k = 20), whatever the distribution, when
// large logits lie anywhere.  Candidates go to shared memory with their ids and are ranked by
// counting.  Rows where that does not work -- NaN, or more ties than the buffer holds -- find the
// exact k-th (logit, id) by bisection instead, over the row as it lies in the cache.
//
// Measured on one B200: 8192 rows of 1024 (fp32, k = 8) 16.3 us, 2.1 TB/s: about 1000 instructions a row, a
// warp each; 160 rows of 128001 (bf16, k = 20) 30.7 us: 148 rows fit at once, and the selection is more than a third.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <float.h>
#include <math.h>
#include <string.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/mossgpu.h"
#include "f32x2.cuh"
#include "op_support.h"

namespace mossgpu {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpMaxTop = 32;
constexpr int kLpMaxCluster = 16;
constexpr int kLpMaxVocab = 500000;
constexpr float kLpLn2 = 0.6931471805599453f, kLpLog2e = 1.4426950408889634f;

struct LpPart {   // what a CTA of a cluster hands to rank 0
    float top, z, s;
    int count;
    unsigned long long best[kLpMaxTop];
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Order-preserving bits of a logit (-0 equals +0); NaN below everything.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return k == 0u ? __int_as_float(0x7fffffff) : __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    return (unsigned long long)order_bits(x) << 32 | uint32_t(~id);
}

// Elements 2 i, 2 i + 1 of a vector, and a vector's largest (NaN if it holds one).
template <typename T>
__device__ __forceinline__ float2 pair_of(const uint4 &v, int i) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    if constexpr (sizeof(T) == 2) {
        if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
}
template <typename T>
__device__ __forceinline__ float largest(const uint4 &v) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
    if constexpr (sizeof(T) == 4) {
        return max_nan(max_nan(__uint_as_float(w[0]), __uint_as_float(w[1])), max_nan(__uint_as_float(w[2]), __uint_as_float(w[3])));
    } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
        const float2 m = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
        return max_nan(m.x, m.y);
    } else {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
        const float2 m = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
        return max_nan(m.x, m.y);
    }
}

// Exact selection of a CTA's first k (logit, id) of its share of a row into `cand`: the order bits
// of the k-th largest by bisection, then the id among its ties.  Returns how many there are.
template <typename T, int NT, typename IdOf>
__device__ __noinline__ int select_exact(const T *x_row, int vocab, int top_k, int vectors, IdOf id_of, int *sum, unsigned long long *cand) {
    constexpr int VE = 16 / int(sizeof(T));
    const auto count = [&](auto &&in) {
        int n = 0;
        for (int v = 0; v < vectors; ++v)
            for (int i = 0; i < VE; ++i) {
                const int id = id_of(v, i);
                if (id >= 0 && id < vocab) n += in(order_bits(float(x_row[id])), id) ? 1 : 0;
            }
        __syncthreads();
        if (threadIdx.x == 0) *sum = 0;
        __syncthreads();
        n = __reduce_add_sync(0xffffffffu, n);
        if ((threadIdx.x & 31) == 0) atomicAdd(sum, n);
        __syncthreads();
        return *sum;
    };
    const int k = min(top_k, count([](uint32_t, int) { return true; }));
    uint32_t key = 0;  // largest key that at least k logits reach
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = key | 1u << bit;
        if (count([=](uint32_t b, int) { return b >= trial; }) >= k) key = trial;
    }
    int last = 0;  // smallest id up to which the ties complete the k
    for (int bit = 19; bit >= 0; --bit) {
        const int trial = last + (1 << bit);  // are the ids below `trial` too few?
        if (count([=](uint32_t b, int id) { return b > key || (b == key && id < trial); }) < k) last = trial;
    }
    __syncthreads();
    if (threadIdx.x == 0) *sum = 0;
    __syncthreads();
    if (k > 0)
        for (int v = 0; v < vectors; ++v)
            for (int i = 0; i < VE; ++i) {
                const int id = id_of(v, i);
                if (id < 0 || id >= vocab) continue;
                const float x = float(x_row[id]);
                const uint32_t b = order_bits(x);
                if (b > key || (b == key && id <= last)) cand[atomicAdd(sum, 1)] = order_key(x, id);
            }
    __syncthreads();
    return *sum;
}

// NT threads hold NV vectors each, those from the eighth on in their own places in shared memory (twice
// as many rows are in flight then as registers alone hold); `ctas` CTAs a row.
template <typename T, int NT, int NV, bool CLUSTER>
__global__ void __launch_bounds__(NT, NT == 32 ? 32 : 1024 / NT) k_token_logprobs(
    const __grid_constant__ mossgpu_logprob_args a, int cluster_ctas, int *status) {
    const int ctas = CLUSTER ? cluster_ctas : 1;
    constexpr int VE = 16 / int(sizeof(T));
    // candidates a CTA ranks; 32 groups of a uniform row give about 130 at k = 32
    constexpr int kCandidates = NT == 32 ? 256 : 512;
    __shared__ __align__(16) float group_top[32];
    __shared__ float2 warp_sums[NT / 32];
    __shared__ unsigned long long cand[kCandidates];
    __shared__ int n_cand;
    __shared__ LpPart parts[CLUSTER ? kLpMaxCluster : 1];
    const int tid = threadIdx.x, lane = tid & 31;
    const int row = CLUSTER ? blockIdx.x / ctas : blockIdx.x, rank = CLUSTER ? blockIdx.x - row * ctas : 0;
    const T *x_row = static_cast<const T *>(a.logits) + int64_t(row) * a.row_stride;
    const int lead = int((reinterpret_cast<uintptr_t>(x_row) / sizeof(T)) % VE);  // elements past a 16-byte boundary
    if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (tid == 0) n_cand = 0;

    // ---- the row; vector v holds elements v VE - lead ..
    constexpr int NR = NV < 8 ? NV : 8;
    extern __shared__ __align__(16) uint4 parked[];  // [NV - 8][NT]
    uint4 x[NR] = {};
    const auto vec = [&](int v) -> uint4 { return v < NR ? x[v] : parked[(v - NR) * NT + tid]; };
    const auto id_of = [=](int v, int i) { return ((v * ctas + rank) * NT + tid) * VE - lead + i; };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int e0 = id_of(v, 0);
        uint4 y;
        if (e0 >= 0 && e0 + VE <= a.vocab) {
            if (v >= NR) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(parked + (v - NR) * NT + tid))),
                             "l"(x_row + e0)
                             : "memory");
                continue;
            }
            y = __ldg(reinterpret_cast<const uint4 *>(x_row + e0));
        } else {
            T e[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) e[i] = e0 + i >= 0 && e0 + i < a.vocab ? x_row[e0 + i] : T(-INFINITY);
            memcpy(&y, e, 16);
        }
        if (v < NR) x[v] = y; else parked[(v - NR) * NT + tid] = y;
    }
    float mine = largest<T>(x[0]);
#pragma unroll
    for (int v = 1; v < NR; ++v) mine = max_nan(mine, largest<T>(x[v]));
    if constexpr (NV > NR) {
        asm volatile("cp.async.wait_all;" ::: "memory");  // a thread reads its own places alone
#pragma unroll
        for (int v = NR; v < NV; ++v) mine = max_nan(mine, largest<T>(vec(v)));
    }
    float group = mine;
#pragma unroll
    for (int o = 1; o < NT / 32; o <<= 1) group = max_nan(group, __shfl_xor_sync(0xffffffffu, group, o));
    if (tid % (NT / 32) == 0) group_top[tid / (NT / 32)] = group;
    __syncthreads();

    // ---- every warp: the CTA's maximum, and the k-th largest of the 32 groups' maxima
    const float g = group_top[lane];
    float top = g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    float bound = INFINITY;
    const bool sound = top == top;
    if (a.top_k > 0 && sound) {
        int above = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float4 q = reinterpret_cast<const float4 *>(group_top)[j];
            above += q.x > g || (q.x == g && 4 * j < lane);
            above += q.y > g || (q.y == g && 4 * j + 1 < lane);
            above += q.z > g || (q.z == g && 4 * j + 2 < lane);
            above += q.w > g || (q.w == g && 4 * j + 3 < lane);
        }
        bound = __shfl_sync(0xffffffffu, g, __ffs(__ballot_sync(0xffffffffu, above == a.top_k - 1)) - 1);
        // ---- candidates: few threads have any
        const bool few = bound == -INFINITY;  // fewer than k groups hold anything: every finite logit, and the first ids
        if (mine >= bound) {
            const float least = few ? -FLT_MAX : bound;
            constexpr int kWords = (NV * VE + 31) / 32;
            uint32_t in[kWords];
#pragma unroll
            for (int w = 0; w < kWords; ++w) in[w] = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint4 y = vec(v);
#pragma unroll
                for (int i = 0; i < VE / 2; ++i) {
                    const float2 f = pair_of<T>(y, i);
                    const int bit = (v * VE + 2 * i) % 32;
                    if (f.x >= least) in[(v * VE) / 32] |= 1u << bit;
                    if (f.y >= least) in[(v * VE) / 32] |= 2u << bit;
                }
            }
            if (few) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int e0 = id_of(v, 0);
                    if (e0 >= a.top_k) continue;
                    for (int i = 0; i < VE; ++i)
                        if (e0 + i >= 0 && e0 + i < a.top_k) in[(v * VE) / 32] |= 1u << ((v * VE) % 32 + i);
                }
            }
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                for (; in[w]; in[w] &= in[w] - 1) {
                    const int e = w * 32 + __ffs(in[w]) - 1, id = id_of(e / VE, e % VE), at = atomicAdd(&n_cand, 1);
                    if (at < kCandidates) cand[at] = order_key(float(x_row[id]), id);
                }
        }
    }

    // ---- sums.  x - M comes first: it is exact at the maximum and rounded relative to itself elsewhere, so that an
    // exponent's error is within 2^-22 of the exponent whatever the sizes of the logits and of 1 / T are (x c - M c as one
    // operation would leave half an ulp of M c in it)
    const float c = kLpLog2e / a.temperature;
    float z = 0.f, s = 0.f;
    const float2 base = make_float2(-top, -top), c2 = make_float2(c, c);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint4 y = vec(v);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            const float2 t = mul2(add2(pair_of<T>(y, i), base), c2);
            // 2^-200 is 0, and 0 * infinity stays out of the sum; without a finite maximum NaN goes the same way
            const float t0 = fmaxf(t.x, -200.f), t1 = fmaxf(t.y, -200.f), e0 = ex2(t0), e1 = ex2(t1);
            z += e0, s = fmaf(e0, t0, s);
            z += e1, s = fmaf(e1, t1, s);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) warp_sums[tid >> 5] = make_float2(z, s);
    __syncthreads();
    int n = n_cand;
    if (a.top_k > 0 && (!sound || n > kCandidates)) n = select_exact<T, NT>(x_row, a.vocab, a.top_k, NV, id_of, &n_cand, cand);

    // ---- the CTA's share
    LpPart *mine_part = &parts[rank];
    if constexpr (CLUSTER) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // rank 0 runs, its shared memory may be written
        mine_part = cg::this_cluster().map_shared_rank(&parts[rank], 0);
    }
    for (int i = tid; i < n; i += NT) {
        const unsigned long long key = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > key;
        if (r < a.top_k) mine_part->best[r] = key;
    }
    if (tid < 32) {
        float2 t = tid < NT / 32 ? warp_sums[tid] : make_float2(0.f, 0.f);
#pragma unroll
        for (int o = NT / 64; o > 0; o >>= 1) {
            t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
            t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        }
        if (tid == 0) {
            mine_part->top = top, mine_part->z = t.x, mine_part->s = t.y;
            mine_part->count = min(n, a.top_k);
        }
    }
    if constexpr (CLUSTER) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank != 0) return;
    } else {
        __syncthreads();
    }

    // ---- rank 0: the row
    float m = parts[0].top, zz = parts[0].z, ss = parts[0].s;
    if constexpr (CLUSTER) {
        for (int r = 1; r < ctas; ++r) m = max_nan(m, parts[r].top);
        zz = ss = 0.f;
        for (int r = 0; r < ctas; ++r) {
            const LpPart &q = parts[r];
            if (q.top == -INFINITY) continue;  // nothing there
            const float t = fmaxf((q.top - m) * c, -200.f), e = ex2(t);  // sums against the part's own maximum
            zz = fmaf(q.z, e, zz);
            ss = fmaf(e, fmaf(q.z, t, q.s), ss);
        }
    }
    const bool empty = m == -INFINITY, bad = !(m < INFINITY);  // NaN or +inf
    const float log_z = log2f(zz), ln_z = log_z * kLpLn2, inv_t = 1.f / a.temperature, nan = __int_as_float(0x7fffffff);
    // (v - m) / T rather than ln 2 t: t of the type's lowest value is past the range of fp32
    // (and where v - m is past it as well, a high temperature may bring it back)
    const auto logprob = [&](float v) {
        if (bad || v == -INFINITY) return bad ? nan : v;
        const float d = v - m;
        return (d == -INFINITY ? fmaf(v, inv_t, -m * inv_t) : d * inv_t) - ln_z;
    };
    if (tid == 0) {
        if (a.logprob) {
            const int t = __ldg(a.tokens + row);
            float lp = 0.f;
            if (t >= a.vocab) {
                lp = nan;
                if (status) atomicCAS(status, 0, kStatusBadToken);
            } else if (t >= 0) {
                lp = logprob(float(x_row[t]));
            }
            a.logprob[row] = lp;
        }
        if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.f : (log_z - ss / zz) * kLpLn2;
    }
    if (a.top_k == 0) return;
    if constexpr (!CLUSTER) {
        for (int i = tid; i < a.top_k; i += NT) {  // a CTA has the whole row: top_k <= vocab entries are there
            const unsigned long long key = parts[0].best[i];
            const int64_t to = int64_t(row) * a.top_k + i;
            if (a.top_ids) a.top_ids[to] = int32_t(~uint32_t(key));
            if (a.top_logprobs) a.top_logprobs[to] = logprob(order_value(uint32_t(key >> 32)));
        }
    } else {
        // merge the parts' sorted lists: an entry's place is its own plus, of every other part, how many are
        // larger.  The largest of the parts' k-th entries bounds the k-th from below, which leaves few.
        __shared__ int place[kLpMaxCluster * kLpMaxTop];
        unsigned long long least = lane < ctas && parts[lane].count >= a.top_k ? parts[lane].best[a.top_k - 1] : 0ull;
#pragma unroll
        for (int o = kLpMaxCluster / 2; o > 0; o >>= 1) least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
        least = __shfl_sync(0xffffffffu, least, 0);
        const int entries = ctas * a.top_k;
        for (int i = tid; i < entries; i += NT) place[i] = i % a.top_k;
        __syncthreads();
        for (int i = tid; i < entries * ctas; i += NT) {
            const int e = i / ctas, q = i - e * ctas, r = e / a.top_k, j = e - r * a.top_k;
            if (q == r || j >= parts[r].count) continue;
            const unsigned long long key = parts[r].best[j];
            if (key < least) continue;
            int lo = 0, hi = parts[q].count;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (parts[q].best[mid] > key) lo = mid + 1; else hi = mid;
            }
            if (lo > 0) atomicAdd(place + e, lo);
        }
        __syncthreads();
        for (int e = tid; e < entries; e += NT) {
            const int r = e / a.top_k, j = e - r * a.top_k;
            if (j >= parts[r].count) continue;
            const unsigned long long key = parts[r].best[j];
            if (key < least || place[e] >= a.top_k) continue;
            const int64_t to = int64_t(row) * a.top_k + place[e];
            if (a.top_ids) a.top_ids[to] = int32_t(~uint32_t(key));
            if (a.top_logprobs) a.top_logprobs[to] = logprob(order_value(uint32_t(key >> 32)));
        }
    }
}

template <typename T, int NT, int NV, bool CLUSTER = false>
cudaError_t launch(const mossgpu_logprob_args &a, int ctas, int *status, cudaStream_t st) {
    auto *kernel = k_token_logprobs<T, NT, NV, CLUSTER>;
    const int smem = NV > 8 ? (NV - 8) * NT * 16 : 0;
    if (smem > 0) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    if (ctas > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(a.rows) * unsigned(ctas));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(ctas);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CLUSTER ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, ctas, status);
}

template <typename T>
cudaError_t dispatch(const mossgpu_logprob_args &a, int *status, cudaStream_t st) {
    // vectors a row touches: one more where rows start off a 16-byte boundary
    constexpr int VE = 16 / int(sizeof(T));
    const bool even = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.row_stride % VE == 0 || a.rows == 1);
    const int n = (a.vocab + (even ? 0 : VE - 1) + VE - 1) / VE;
    // Two or four vectors a thread where all rows' threads are resident at once: a row's latency is what its
    // longest thread does (one row of 128001 logits: 10.8 us against 14.8 with 16 vectors, 12.9 on 16 CTAs).
    // More otherwise: the per-row work is spread over more logits (160 such rows: 30 us against 41 with four).
    const int64_t threads = int64_t(148) * 1024;
    if (int64_t(a.rows) * n <= 2 * threads) {
        if (n <= 2 * 128) return launch<T, 128, 2>(a, 1, status, st);
        if (n <= 2 * 512) return launch<T, 512, 2>(a, 1, status, st);
        for (int ctas = 2; ctas <= 8; ctas *= 2)
            if (n <= 2 * 512 * ctas) return launch<T, 512, 2, true>(a, ctas, status, st);
        if (n <= 4 * 512 * 8) return launch<T, 512, 4, true>(a, 8, status, st);
    }
    if (n <= 8 * 32) return launch<T, 32, 8>(a, 1, status, st);
    if (n <= 8 * 128) return launch<T, 128, 8>(a, 1, status, st);
    if (n <= 8 * 512) return launch<T, 512, 8>(a, 1, status, st);
    if (n <= 16 * 512) return launch<T, 512, 16>(a, 1, status, st);
    int ctas = 2;
    while (ctas < kLpMaxCluster && n > 16 * 512 * ctas) ctas *= 2;
    return launch<T, 512, 16, true>(a, ctas, status, st);
}

}  // namespace
}  // namespace mossgpu

extern "C" int mossgpu_token_logprobs(const mossgpu_logprob_args *args, void *cuda_stream) {
    using namespace mossgpu;
    const char *who = "token_logprobs";
    if (!args) return op_errorf("%s: args is NULL", who);
    const mossgpu_logprob_args &a = *args;
    if (a.rows < 0 || a.rows > (1 << 26)) return op_errorf("%s: rows = %d must be 0 .. 2^26", who, a.rows);
    if (a.vocab < 1 || a.vocab > kLpMaxVocab) return op_errorf("%s: vocab = %d must be 1 .. %d", who, a.vocab, kLpMaxVocab);
    if (a.type < MOSSGPU_F32 || a.type > MOSSGPU_BF16) return op_errorf("%s: type %d is no element type", who, a.type);
    if (a.top_k < 0 || a.top_k > kLpMaxTop || a.top_k > a.vocab)
        return op_errorf("%s: top_k = %d must be 0 .. min(%d, vocab)", who, a.top_k, kLpMaxTop);
    if (!(a.temperature > 0.f) || !(a.temperature < INFINITY) || !(kLpLog2e / a.temperature < INFINITY))
        return op_errorf("%s: temperature must be positive, and it and log2(e) / temperature finite", who);
    if (a.rows > 1 && a.row_stride < a.vocab) return op_errorf("%s: row_stride is below vocab", who);
    if (a.rows == 0) return 0;
    if (!a.logits) return op_errorf("%s: logits is NULL", who);
    if ((a.logprob != nullptr) != (a.tokens != nullptr)) return op_errorf("%s: tokens and logprob come together", who);
    if (a.top_k > 0 && !a.top_ids && !a.top_logprobs) return op_errorf("%s: top_k without top_ids or top_logprobs", who);
    if (a.top_k == 0 && (a.top_ids || a.top_logprobs)) return op_errorf("%s: top_ids or top_logprobs without top_k", who);
    if (!a.logprob && !a.entropy && a.top_k == 0) return op_errorf("%s: nothing is asked for", who);
    const size_t size = a.type == MOSSGPU_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a.logits) % size != 0) return op_errorf("%s: logits is not aligned to its type", who);
    for (const void *p : {static_cast<const void *>(a.tokens), static_cast<const void *>(a.logprob), static_cast<const void *>(a.entropy),
                          static_cast<const void *>(a.top_ids), static_cast<const void *>(a.top_logprobs)})
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return op_errorf("%s: a pointer is not aligned to its type", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = a.type == MOSSGPU_F32   ? dispatch<float>(a, status, st)
                          : a.type == MOSSGPU_F16 ? dispatch<__half>(a, status, st)
                                                  : dispatch<__nv_bfloat16>(a, status, st);
    return e == cudaSuccess ? 0 : op_errorf("%s launch: %s", who, cudaGetErrorString(e));
}
