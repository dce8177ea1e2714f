// logprob.cu -- log-probabilities of given tokens, entropy and the most likely tokens of rows of
// logits (mossgpu_token_logprobs).
//
// A row is held in registers, 32 logits a thread, by one CTA of 32 to 1024 threads or by a
// cluster of up to 16: it is read from HBM once, and the maximum, the sums and the selection all
// work on what was read.  With x the logits, c = log2(e) / T and M = max x:
//   Z = sum 2^((x - M) c),  S = sum 2^((x - M) c) (x - M),
//   log p_t = (x_t - M) / T - ln Z,  entropy = ln Z - S / (T Z).
// CTAs of a cluster sum against their own maxima; rank 0 merges.
//
// Selection: the threads form 32 groups; the k-th largest of the groups' maxima bounds the k-th
// largest logit from below, so only logits from it on are candidates: for k of 32 groups about
// -32 ln(1 - k / 32) are expected (9 for k = 8, 31 for k = 20), whatever the distribution, when
// large logits lie anywhere.  Candidates go to shared memory with their ids and are ranked by
// counting.  Rows where that does not work -- NaN, or more ties than the buffer holds -- find the
// exact k-th (logit, id) by bisection instead.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <math.h>

#include "../../include/mossgpu.h"
#include "op_support.h"

namespace mossgpu {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpPerThread = 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxCluster = 16;
constexpr int kLpMaxVocab = 500000;

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

// Order-preserving bits of a logit; NaN below everything.  (-0 was made +0 when it was read.)
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return k == 0u ? __int_as_float(0x7fffffff) : __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == 32 ? 24 : 1024 / NT) k_token_logprobs(const __grid_constant__ mossgpu_logprob_args a, int ctas, int *status) {
    constexpr int VE = 16 / int(sizeof(T));
    constexpr int NV = kLpPerThread / VE;
    __shared__ __align__(16) float group_top[32];
    __shared__ float2 warp_sums[NT / 32];
    // candidates a CTA ranks; 32 groups of a uniform row give about 130 at k = 32
    constexpr int kLpCandidates = NT == 32 ? 256 : 512;
    __shared__ unsigned long long cand[kLpCandidates];
    __shared__ int n_cand, n_cand_old;
    __shared__ LpPart parts[NT < 512 ? 1 : kLpMaxCluster];  // clusters have CTAs of 512 threads or more
    const int tid = threadIdx.x, lane = tid & 31;
    const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas;
    const T *x_row = static_cast<const T *>(a.logits) + int64_t(row) * a.row_stride;
    const int lead = int((reinterpret_cast<uintptr_t>(x_row) / sizeof(T)) % VE);  // elements past a 16-byte boundary
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (tid == 0) n_cand = 0;

    // ---- the row; vector v holds elements v VE - lead ..
    float x[NV][VE];
    const auto id_of = [&](int v, int i) { return ((v * ctas + rank) * NT + tid) * VE - lead + i; };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int e0 = id_of(v, 0);
        if (e0 >= 0 && e0 + VE <= a.vocab) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(x_row + e0));
            const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int i = 0; i < VE; ++i) x[v][i] = float(e[i]) + 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i)
                x[v][i] = e0 + i >= 0 && e0 + i < a.vocab ? float(x_row[e0 + i]) + 0.f : -INFINITY;
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < VE; ++i) mine = max_nan(mine, x[v][i]);
#pragma unroll
    for (int o = 1; o < NT / 32; o <<= 1) mine = max_nan(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (tid % (NT / 32) == 0) group_top[tid / (NT / 32)] = mine;
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
    }

    // ---- sums, and candidates
    float z = 0.f, s = 0.f;
    const float c = 1.4426950408889634f / a.temperature;
    const bool few = bound == -INFINITY;  // fewer than k groups hold anything: every finite logit, and the first ids
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const float d = x[v][i] - top;
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * c));
            z += e;
            s = fmaf(e, fmaxf(d, -3e38f), s);  // 0 * infinity stays out of the sum
        }
    if (a.top_k > 0 && sound) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                bool in = x[v][i] >= bound;
                if (few) {
                    const int id = id_of(v, i);
                    in = id >= 0 && id < a.vocab && (x[v][i] > -INFINITY || id < a.top_k);
                }
                if (in) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kLpCandidates)
                        cand[at] = (unsigned long long)order_bits(x[v][i]) << 32 | uint32_t(~id_of(v, i));
                }
            }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) warp_sums[tid >> 5] = make_float2(z, s);
    __syncthreads();

    if (a.top_k > 0 && (!sound || n_cand > kLpCandidates)) {
        // ---- exact selection: bisect the order bits of the k-th largest, then the id among its ties
        int valid = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < VE; ++i) valid += id_of(v, i) >= 0 && id_of(v, i) < a.vocab;
        const auto block_sum = [&](int n) {
            __syncthreads();
            if (tid == 0) n_cand_old = 0;
            __syncthreads();
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) atomicAdd(&n_cand_old, n);
            __syncthreads();
            return n_cand_old;
        };
        const int k = min(a.top_k, block_sum(valid));
        uint32_t key = 0;  // largest key that at least k logits reach
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = key | 1u << bit;
            int n = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    n += order_bits(x[v][i]) >= trial && id_of(v, i) >= 0 && id_of(v, i) < a.vocab;
            if (block_sum(n) >= k) key = trial;
        }
        int last = 0;  // smallest id up to which the ties complete the k
        for (int bit = 19; bit >= 0; --bit) {
            const int trial = last + (1 << bit);  // are the ids below `trial` too few?
            int n = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const int id = id_of(v, i);
                    const uint32_t b = order_bits(x[v][i]);
                    n += id >= 0 && id < a.vocab && (b > key || (b == key && id < trial));
                }
            if (block_sum(n) < k) last = trial;
        }
        __syncthreads();
        if (tid == 0) n_cand = 0;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const int id = id_of(v, i);
                const uint32_t b = order_bits(x[v][i]);
                if (k > 0 && id >= 0 && id < a.vocab && (b > key || (b == key && id <= last)))
                    cand[atomicAdd(&n_cand, 1)] = (unsigned long long)b << 32 | uint32_t(~id);
            }
        __syncthreads();
    }

    // ---- the CTA's share
    LpPart *mine_part = &parts[rank];
    if (ctas > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // rank 0 runs, its shared memory may be written
        mine_part = cg::this_cluster().map_shared_rank(&parts[rank], 0);
    }
    const int n = min(n_cand, kLpCandidates);
    for (int i = tid; i < n; i += NT) {
        const unsigned long long key = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > key;
        if (r < a.top_k) mine_part->best[r] = key;
    }
    if (tid < 32) {
        float2 t = tid < NT / 32 ? warp_sums[tid] : make_float2(0.f, 0.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
            t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        }
        if (tid == 0) mine_part->top = top, mine_part->z = t.x, mine_part->s = t.y, mine_part->count = min(n, a.top_k);
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank != 0) return;
    } else {
        __syncthreads();
    }

    // ---- rank 0: the row
    float m = -INFINITY;
    for (int r = 0; r < ctas; ++r) m = max_nan(m, parts[r].top);
    float zz = 0.f, ss = 0.f;
    for (int r = 0; r < ctas; ++r) {
        const LpPart &q = parts[r];
        if (q.top == -INFINITY) continue;  // nothing there
        const float d = q.top - m;         // sums against the part's own maximum
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * c));
        zz = fmaf(q.z, e, zz);
        ss = fmaf(e, fmaf(q.z, fmaxf(d, -1e30f), q.s), ss);
    }
    const float inv_t = 1.f / a.temperature;
    const bool empty = m == -INFINITY, bad = !(m < INFINITY);  // NaN or +inf
    const float ln_z = logf(zz), nan = __int_as_float(0x7fffffff);
    const auto logprob = [&](float v) { return bad ? nan : v == -INFINITY ? -INFINITY : (v - m) * inv_t - ln_z; };
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
        if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.f : ln_z - ss / zz * inv_t;
    }
    if (a.top_k > 0) {
        // merge the parts' sorted lists: an entry's rank is its own plus, of every other part, how many are larger
        for (int i = tid; i < ctas * kLpMaxTop; i += NT) {
            const int r = i / kLpMaxTop, j = i % kLpMaxTop;
            if (j >= parts[r].count) continue;
            const unsigned long long key = parts[r].best[j];
            int at = j;
            for (int q = 0; q < ctas; ++q) {
                if (q == r) continue;
                int lo = 0, hi = parts[q].count;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (parts[q].best[mid] > key) lo = mid + 1; else hi = mid;
                }
                at += lo;
            }
            if (at < a.top_k) {
                const int64_t to = int64_t(row) * a.top_k + at;
                if (a.top_ids) a.top_ids[to] = int32_t(~uint32_t(key));
                if (a.top_logprobs) a.top_logprobs[to] = logprob(order_value(uint32_t(key >> 32)));
            }
        }
    }
}

template <typename T, int NT>
cudaError_t launch(const mossgpu_logprob_args &a, int ctas, int *status, cudaStream_t st) {
    auto *kernel = k_token_logprobs<T, NT>;
    if (ctas > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(a.rows) * unsigned(ctas));
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(ctas);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, ctas, status);
}

template <typename T>
cudaError_t dispatch(const mossgpu_logprob_args &a, int *status, cudaStream_t st) {
    // threads a row needs at 32 logits each, one vector more where rows start off a 16-byte boundary
    constexpr int VE = 16 / int(sizeof(T));
    const int need = (a.vocab + VE - 1 + kLpPerThread - 1) / kLpPerThread;
    if (need <= 32 || (a.vocab <= 1024 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.row_stride % VE == 0))
        return launch<T, 32>(a, 1, status, st);
    if (need <= 128) return launch<T, 128>(a, 1, status, st);
    if (need <= 512) return launch<T, 512>(a, 1, status, st);
    int ctas = 2;
    while (ctas < 8 && need > 512 * ctas) ctas *= 2;
    if (need <= 512 * ctas) return launch<T, 512>(a, ctas, status, st);
    while (ctas < kLpMaxCluster && need > 1024 * ctas) ctas *= 2;
    return launch<T, 1024>(a, ctas, status, st);
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
    if (!(a.temperature > 0.f) || !(a.temperature < INFINITY) || !(1.f / a.temperature < INFINITY))
        return op_errorf("%s: temperature must be positive, and it and its inverse finite", who);
    if (a.rows > 1 && a.row_stride < a.vocab) return op_errorf("%s: row_stride is below vocab", who);
    if (a.rows == 0) return 0;
    if (!a.logits) return op_errorf("%s: logits is NULL", who);
    if ((a.logprob != nullptr) != (a.tokens != nullptr)) return op_errorf("%s: tokens and logprob come together", who);
    if (a.top_k > 0 && !a.top_ids && !a.top_logprobs) return op_errorf("%s: top_k without top_ids or top_logprobs", who);
    if (a.top_k == 0 && (a.top_ids || a.top_logprobs)) return op_errorf("%s: top_ids or top_logprobs without top_k", who);
    if (!a.logprob && !a.entropy && a.top_k == 0) return op_errorf("%s: nothing is asked for", who);
    const size_t size = a.type == MOSSGPU_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a.logits) % size != 0) return op_errorf("%s: logits is not aligned to its type", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = a.type == MOSSGPU_F32   ? dispatch<float>(a, status, st)
                          : a.type == MOSSGPU_F16 ? dispatch<__half>(a, status, st)
                                                  : dispatch<__nv_bfloat16>(a, status, st);
    return e == cudaSuccess ? 0 : op_errorf("%s launch: %s", who, cudaGetErrorString(e));
}
