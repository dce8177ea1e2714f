// kv8.cu -- C entry points of the rotary and 8-bit-cache operators (kernels: rope_kv8.cuh,
// attn_kv8.cuh; the index checks: kv8_index.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "attn_kv8.cuh"
#include "types.h"

namespace mossgpu {
namespace {

constexpr int kMaxHeads = 1 << 30;  // the kernels' head counters step past the last head by at most 2^18

size_t type_size(int type) { return type == MOSSGPU_F32 ? 4 : 2; }
bool is_type(int type) { return type >= MOSSGPU_F32 && type <= MOSSGPU_BF16; }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Accesses of `bytes` at every head's multiples of them
bool vec_ok(const void *p, int64_t row, int64_t head, int type, size_t bytes) {
    const int64_t e = int64_t(bytes / type_size(type));
    return aligned(p, bytes) && row % e == 0 && head % e == 0;
}
// 8 elements
bool vec8_ok(const void *p, int64_t row, int64_t head, int type) { return vec_ok(p, row, head, type, 8 * type_size(type)); }

int check_cache(const mossgpu_kv8_cache *c, const char *who) {
    if (!c) return op_errorf("%s: cache is NULL", who);
    if (!c->codes || !c->scales || !c->page_table) return op_errorf("%s: a pointer of the cache is NULL", who);
    if (!aligned(c->codes, 16) || !aligned(c->scales, 16)) return op_errorf("%s: codes and scales must be 16-byte aligned", who);
    if (!aligned(c->page_table, 4)) return op_errorf("%s: page_table is not aligned to its type", who);
    if (c->n_pages < 1 || c->n_slots < 1 || c->pages_per_slot < 1)
        return op_errorf("%s: n_pages, n_slots and pages_per_slot must be positive", who);
    if (c->pages_per_slot > (1 << 26)) return op_errorf("%s: pages_per_slot is above 2^26", who);
    if (c->kv_heads < 1 || c->kv_heads > 1024) return op_errorf("%s: kv_heads = %d must be 1 .. 1024", who, c->kv_heads);
    if (c->head_dim != 64 && c->head_dim != 128) return op_errorf("%s: head_dim = %d must be 64 or 128", who, c->head_dim);
    if (c->format != MOSSGPU_KV_INT8 && c->format != MOSSGPU_KV_E4M3) return op_errorf("%s: format %d is none", who, c->format);
    return 0;
}

// 1: refused, -1: nothing to do
int check_seqs(const mossgpu_seq_batch *s, const char *who) {
    if (!s) return op_errorf("%s: seqs is NULL", who);
    if (s->n_seqs < 0 || s->n_seqs > kAk8MaxSeqs) return op_errorf("%s: n_seqs = %d must be 0 .. %d", who, s->n_seqs, kAk8MaxSeqs);
    if (s->rows < 0) return op_errorf("%s: rows = %d is negative", who, s->rows);
    if (s->n_seqs == 0 || s->rows == 0) return -1;
    if (!s->row_start || !s->slot || !s->ctx_len) return op_errorf("%s: a pointer of seqs is NULL", who);
    if (!aligned(s->row_start, 4) || !aligned(s->slot, 4) || !aligned(s->ctx_len, 4))
        return op_errorf("%s: a pointer of seqs is not aligned to its type", who);
    return 0;
}

int check_rope(const mossgpu_rope *r, int head_dim, const char *who) {
    if (!r->steps) return op_errorf("%s: steps is NULL", who);
    if (!aligned(r->steps, 8)) return op_errorf("%s: steps is not aligned to its type", who);
    if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > head_dim)
        return op_errorf("%s: rotary_dim = %d must be even, 2 .. head_dim", who, r->rotary_dim);
    if (!std::isfinite(r->magnitude)) return op_errorf("%s: magnitude is not finite", who);
    return 0;
}

// A [rows][heads][head_dim] tensor that is written: its heads may not overlap.
bool distinct(int rows, int heads, int head_dim, int64_t row, int64_t head) {
    if (row < 0 || head < 0) return false;
    if (heads > 1 && head < head_dim) return rows > 1 ? row >= head_dim && head >= row * (rows - 1) + head_dim : false;
    if (rows > 1 && row < head * (heads - 1) + head_dim) return heads > 1 && row >= head_dim && head >= row * (rows - 1) + head_dim;
    return true;
}

// Warps that share a row (or a few rows) of `passes` passes: one where the rows alone fill the
// machine, as many as there are passes where they do not.
int warps_for(int64_t rows, int passes) {
    const int64_t want = int64_t(kNumSMs) * 24;  // resident at once
    return int(std::max<int64_t>(1, std::min<int64_t>(passes, want / rows)));
}
unsigned blocks_for(int64_t warps) { return unsigned((warps + kRowThreads / 32 - 1) / (kRowThreads / 32)); }

template <typename T, int LAYOUT>
cudaError_t launch_rope(RowOp a, cudaStream_t st) {
    const int lanes = a.head_dim <= 32 ? 4 : a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32, heads = 32 / lanes;
    a.row_warps = warps_for(a.rows, (a.heads[0] + heads - 1) / heads + 2 * ((a.heads[1] + heads - 1) / heads));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_for(int64_t(a.rows) * a.row_warps));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = st;
    if (a.heads[1] > 0)
        return lanes == 8 ? cudaLaunchKernelEx(&cfg, k_rope_append<T, 8, LAYOUT, true>, a)
                          : cudaLaunchKernelEx(&cfg, k_rope_append<T, 16, LAYOUT, true>, a);
    if (lanes == 4) return cudaLaunchKernelEx(&cfg, k_rope_append<T, 4, LAYOUT, false>, a);
    if (lanes == 8) return cudaLaunchKernelEx(&cfg, k_rope_append<T, 8, LAYOUT, false>, a);
    if (lanes == 16) return cudaLaunchKernelEx(&cfg, k_rope_append<T, 16, LAYOUT, false>, a);
    return cudaLaunchKernelEx(&cfg, k_rope_append<T, 32, LAYOUT, false>, a);
}

int run_rope(const RowOp &a, int type, bool vec, void *stream, const char *who) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int layout = !vec ? kAny : a.rope.rotary_dim == 0 || a.rope.interleaved ? kPairs : a.rope.rotary_dim % 8 == 0 ? kHalves : kAny;
    const auto of = [&](auto zero) {
        using T = decltype(zero);
        return layout == kPairs ? launch_rope<T, kPairs>(a, st) : layout == kHalves ? launch_rope<T, kHalves>(a, st) : launch_rope<T, kAny>(a, st);
    };
    const cudaError_t e = type == MOSSGPU_F32 ? of(float()) : type == MOSSGPU_F16 ? of(__half()) : of(__nv_bfloat16());
    return e == cudaSuccess ? 0 : op_errorf("%s launch: %s", who, cudaGetErrorString(e));
}

template <typename T>
cudaError_t launch_read(ReadOp a, cudaStream_t st) {
    const int rows = a.cache.head_dim == 64 ? 16 : 8;  // of a warp
    const int64_t groups = (int64_t(a.seqs.rows) + rows - 1) / rows;
    a.row_warps = warps_for(groups, 2 * a.cache.kv_heads);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_for(groups * a.row_warps));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = st;
    return a.cache.head_dim == 64 ? cudaLaunchKernelEx(&cfg, k_kv8_read<T, 64>, a) : cudaLaunchKernelEx(&cfg, k_kv8_read<T, 128>, a);
}

// ---- attention ---------------------------------------------------------------------------


// The kernel of a call: which form, and what it needs.
struct AttnForm {
    void (*kernel)(AttnKv8);
    int warps, ctas, ring, tile_rows;  // ctas: of an SM
    int runs;                          // warps or CTAs that take a run each; 0: a CTA has a whole unit (one launch)
};

template <int D, int FORMAT, int MODE>
AttnForm attn_rows(int64_t rows_per_unit, bool direct) {
    using S = Ak8Shape<D>;
    using B = Ak8Block<D>;
    constexpr int kRows = Rows<D, MODE>::kRows;
    if (direct) return {k_attn_kv8<D, FORMAT, MODE, true>, S::kWarps, 1, S::kRing, kRows, 0};
    // A warp a unit reads and converts a tile again for every 8 or 16 rows, a CTA once for 32 or 64, but takes as
    // long for few of them.  48 sequences of 700-8000 positions, 8 kv heads of 128, e4m3, bf16 (us when repeated for a
    // second; warp, CTA): 20 rows 212, 252; 32 rows 224, 258; 48 rows 324, 296; 64 rows 430, 320; 96 rows 626, 555.
    // The other types, sizes and formats go by the same count of rows a product, unmeasured.
    if (rows_per_unit <= 2 * kRows) return {k_attn_kv8<D, FORMAT, MODE, false>, S::kWarps, 1, S::kRing, kRows, kNumSMs * S::kWarps};
    return {k_attn_kv8_block<D, FORMAT, MODE>, B::kWarps, B::kCtas, B::kRing, B::kWarps * kRows, kNumSMs * B::kCtas};
}

template <int D, int FORMAT>
AttnForm attn_form(int type, int64_t rows_per_unit, int64_t rows, int n_seqs, int kv_heads, int pages) {
    // A CTA a unit (one launch) where that is few rounds of CTAs and no warp gets more than 8 tiles of 32
    // positions, which is known by the width of the table alone.  Us, one launch against two, 12 heads of 64: one stream
    // of 300 positions 7.0, 10.8; 8 x 1000 8.3, 16.5; 32 x 1000 (480 units) 20.6, 24.6; but 32 x 100-3000 27.1, 26.8,
    // and one of 4000 16.5, 14.4.
    const auto direct = [&](int tile_rows, int warps) { return (rows / tile_rows + n_seqs) * kv_heads <= 4 * kNumSMs && pages <= 2 * 8 * warps; };
    // The form for 4 rows takes 8 in two units.  Streams of 256-4096 positions, 12 kv heads of 64, int8, fp32 (us when
    // repeated for a second; this form, the next, on one card): one row of 512 streams 345, 386; 4 rows of 128 streams
    // 98, 109; 8 rows 180, 114.
    if (rows_per_unit <= 4) {
        using S = Ak8Few<D>;
        if (direct(4, S::kWarps)) return {k_attn_kv8_few<D, FORMAT, true>, S::kWarps, 1, S::kRing, 4, 0};
        return {k_attn_kv8_few<D, FORMAT, false>, S::kWarps, 1, S::kRing, 4, kNumSMs * S::kWarps};
    }
    const bool one = direct(type == MOSSGPU_BF16 ? 16 : 8, Ak8Shape<D>::kWarps);
    if (type != MOSSGPU_BF16) return attn_rows<D, FORMAT, kSplit>(rows_per_unit, one);
    return attn_rows<D, FORMAT, kHalf>(rows_per_unit, one);
}

// Mean query rows of a sequence and kv head decide: the forms differ in speed, not in what they can do.
AttnForm attn_form(const mossgpu_kv8_cache &c, int type, int64_t rows, int n_seqs, int group) {
    const int64_t per_unit = (rows + n_seqs - 1) / n_seqs * group;
    const auto form = c.head_dim == 64 ? (c.format == MOSSGPU_KV_INT8 ? attn_form<64, MOSSGPU_KV_INT8> : attn_form<64, MOSSGPU_KV_E4M3>)
                                       : (c.format == MOSSGPU_KV_INT8 ? attn_form<128, MOSSGPU_KV_INT8> : attn_form<128, MOSSGPU_KV_E4M3>);
    return form(type, per_unit, rows * group, n_seqs, c.kv_heads, c.pages_per_slot);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t plan_bytes() { return round256(sizeof(uint32_t) * (2 * kAk8MaxSeqs + 1)); }

// Enough for every form: two partials a run and head
size_t workspace_of(int head_dim, int kv_heads, int64_t rows_in_unit) {
    const size_t row = size_t(head_dim + 4) * sizeof(float);
    const int64_t few = kNumSMs * (head_dim == 64 ? Ak8Few<64>::kWarps : Ak8Few<128>::kWarps) * std::min<int64_t>(4, rows_in_unit);
    const int64_t warp = kNumSMs * (head_dim == 64 ? Ak8Shape<64>::kWarps : Ak8Shape<128>::kWarps) * std::min<int64_t>(16, rows_in_unit);
    const int64_t block = std::max<int64_t>(kNumSMs * Ak8Block<64>::kCtas, kv_heads) * std::min<int64_t>(64, rows_in_unit);
    return plan_bytes() + 2 * size_t(std::max(few, std::max(warp, block))) * row;
}

}  // namespace
}  // namespace mossgpu

using namespace mossgpu;

extern "C" {

int mossgpu_rope_steps(int rotary_dim, double base, const mossgpu_rope_scaling *scaling, uint64_t *steps, float *magnitude) {
    const char *who = "rope_steps";
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > kMaxRopeDim)
        return op_errorf("%s: rotary_dim = %d must be even, 2 .. %d", who, rotary_dim, kMaxRopeDim);
    if (!(base > 1.0) || !std::isfinite(base)) return op_errorf("%s: base must be finite and above 1", who);
    if (!steps) return op_errorf("%s: steps is NULL", who);
    const int kind = scaling ? scaling->kind : 0;
    if (kind < 0 || kind > 3) return op_errorf("%s: scaling kind %d is none", who, kind);
    const double factor = kind ? scaling->factor : 1.0;
    if (!(factor >= 1.0) || !std::isfinite(factor)) return op_errorf("%s: factor must be finite, 1 or above", who);
    if (kind == 2 && rotary_dim == 2) return op_errorf("%s: base scaling needs a rotary_dim above 2", who);
    if (kind == 3 && (!(scaling->original_len > 0.0) || !std::isfinite(scaling->original_len) || !(scaling->slow >= 0.0) ||
                      !(scaling->fast > scaling->slow) || !std::isfinite(scaling->fast)))
        return op_errorf("%s: the ramp needs original_len > 0 and 0 <= slow < fast", who);
    if (kind == 2) base *= std::pow(factor, double(rotary_dim) / double(rotary_dim - 2));
    const double two_pi = 6.283185307179586476925286766559;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (kind == 1) f /= factor;
        if (kind == 3) {
            const double turns = scaling->original_len * f / two_pi;
            const double keep = std::min(1.0, std::max(0.0, (turns - scaling->slow) / (scaling->fast - scaling->slow)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        steps[i] = uint64_t(std::nearbyint(std::ldexp(f / two_pi, 64)));  // f <= 1: below 2^62
    }
    if (magnitude) *magnitude = kind == 3 ? float(0.1 * std::log(factor) + 1.0) : 1.f;
    return 0;
}

int mossgpu_rope_rotate(const mossgpu_rope *rope, const mossgpu_rope_args *args, void *cuda_stream) {
    const char *who = "rope_rotate";
    if (!rope || !args) return op_errorf("%s: a descriptor is NULL", who);
    const mossgpu_rope_args &g = *args;
    if (g.rows < 0 || g.heads < 0) return op_errorf("%s: rows and heads must not be negative", who);
    if (g.heads > kMaxHeads) return op_errorf("%s: heads = %d is above 2^30", who, g.heads);
    if (g.head_dim < 8 || g.head_dim > kMaxRopeDim || g.head_dim % 8)
        return op_errorf("%s: head_dim = %d must be a multiple of 8, 8 .. %d", who, g.head_dim, kMaxRopeDim);
    if (!is_type(g.type)) return op_errorf("%s: type %d is no element type", who, g.type);
    if (check_rope(rope, g.head_dim, who) != 0) return 1;
    if (g.rows == 0 || g.heads == 0) return 0;
    if (!g.x || !g.out || !g.pos) return op_errorf("%s: a required pointer is NULL", who);
    if (!aligned(g.x, type_size(g.type)) || !aligned(g.out, type_size(g.type)) || !aligned(g.pos, 4))
        return op_errorf("%s: a pointer is not aligned to its type", who);
    if (!distinct(g.rows, g.heads, g.head_dim, g.out_row_stride, g.out_head_stride))
        return op_errorf("%s: the strides of out make its heads overlap", who);
    if (g.x == g.out && (g.x_row_stride != g.out_row_stride || g.x_head_stride != g.out_head_stride))
        return op_errorf("%s: in place, x and out must have the same strides", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    RowOp a{};
    a.rope = *rope;
    a.src[0] = g.x;
    a.q_out = g.out;
    a.row_stride[0] = g.x_row_stride, a.head_stride[0] = g.x_head_stride;
    a.out_row_stride = g.out_row_stride, a.out_head_stride = g.out_head_stride;
    a.pos = g.pos;
    a.heads[0] = g.heads;
    const bool vec = vec8_ok(g.x, g.x_row_stride, g.x_head_stride, g.type) && vec8_ok(g.out, g.out_row_stride, g.out_head_stride, g.type);
    a.rows = g.rows;
    a.head_dim = g.head_dim;
    a.inverse = g.inverse;
    a.status = status;
    return run_rope(a, g.type, vec, cuda_stream, who);
}

int mossgpu_kv8_append(const mossgpu_kv8_cache *cache, const mossgpu_seq_batch *seqs, const mossgpu_rope *rope,
                       const mossgpu_kv8_append_args *args, void *cuda_stream) {
    const char *who = "kv8_append";
    if (check_cache(cache, who) != 0) return 1;
    const int batch = check_seqs(seqs, who);
    if (batch > 0) return 1;
    if (!args) return op_errorf("%s: args is NULL", who);
    const mossgpu_kv8_append_args &g = *args;
    if (!is_type(g.type)) return op_errorf("%s: type %d is no element type", who, g.type);
    if (rope && check_rope(rope, cache->head_dim, who) != 0) return 1;
    if (g.q && !rope) return op_errorf("%s: q is given without a rope", who);
    if (g.q_heads < 0 || (g.q && g.q_heads == 0)) return op_errorf("%s: q_heads = %d", who, g.q_heads);
    if (g.q_heads > kMaxHeads) return op_errorf("%s: q_heads = %d is above 2^30", who, g.q_heads);
    if (batch < 0) return 0;
    if (!g.k || !g.v || (g.q && !g.q_out)) return op_errorf("%s: a required pointer is NULL", who);
    const size_t size = type_size(g.type);
    if (!aligned(g.k, size) || !aligned(g.v, size) || !aligned(g.q, size) || !aligned(g.q_out, size) || !aligned(g.pos, 4))
        return op_errorf("%s: a pointer is not aligned to its type", who);
    if (g.q && !distinct(seqs->rows, g.q_heads, cache->head_dim, g.q_out_row_stride, g.q_out_head_stride))
        return op_errorf("%s: the strides of q_out make its heads overlap", who);
    if (g.q && g.q == g.q_out && (g.q_row_stride != g.q_out_row_stride || g.q_head_stride != g.q_out_head_stride))
        return op_errorf("%s: in place, q and q_out must have the same strides", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    RowOp a{};
    a.cache = *cache;
    a.seqs = *seqs;
    if (rope) a.rope = *rope;
    a.src[0] = g.q, a.src[1] = g.k, a.src[2] = g.v;
    a.q_out = g.q_out;
    a.row_stride[0] = g.q_row_stride, a.row_stride[1] = g.k_row_stride, a.row_stride[2] = g.v_row_stride;
    a.head_stride[0] = g.q_head_stride, a.head_stride[1] = g.k_head_stride, a.head_stride[2] = g.v_head_stride;
    a.out_row_stride = g.q_out_row_stride, a.out_head_stride = g.q_out_head_stride;
    a.pos = g.pos;
    a.heads[0] = g.q ? g.q_heads : 0;
    a.heads[1] = cache->kv_heads;
    bool vec = !g.q || vec8_ok(g.q_out, g.q_out_row_stride, g.q_out_head_stride, g.type);
    for (int i = g.q ? 0 : 1; i < 3; ++i) vec = vec && vec8_ok(a.src[i], a.row_stride[i], a.head_stride[i], g.type);
    a.rows = seqs->rows;
    a.head_dim = cache->head_dim;
    a.status = status;
    return run_rope(a, g.type, vec, cuda_stream, who);
}

int mossgpu_kv8_read(const mossgpu_kv8_cache *cache, const mossgpu_seq_batch *seqs, const mossgpu_kv8_read_args *args,
                     void *cuda_stream) {
    const char *who = "kv8_read";
    if (check_cache(cache, who) != 0) return 1;
    const int batch = check_seqs(seqs, who);
    if (batch > 0) return 1;
    if (!args) return op_errorf("%s: args is NULL", who);
    const mossgpu_kv8_read_args &g = *args;
    if (!is_type(g.type)) return op_errorf("%s: type %d is no element type", who, g.type);
    if (batch < 0) return 0;
    if (!g.k && !g.v) return op_errorf("%s: k and v are both NULL", who);
    if (!aligned(g.k, type_size(g.type)) || !aligned(g.v, type_size(g.type)))
        return op_errorf("%s: a pointer is not aligned to its type", who);
    if ((g.k && !distinct(seqs->rows, cache->kv_heads, cache->head_dim, g.k_row_stride, g.k_head_stride)) ||
        (g.v && !distinct(seqs->rows, cache->kv_heads, cache->head_dim, g.v_row_stride, g.v_head_stride)))
        return op_errorf("%s: the strides of an output make its heads overlap", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    ReadOp a{};
    a.cache = *cache;
    a.seqs = *seqs;
    a.out[0] = g.k, a.out[1] = g.v;
    a.row_stride[0] = g.k_row_stride, a.row_stride[1] = g.v_row_stride;
    a.head_stride[0] = g.k_head_stride, a.head_stride[1] = g.v_head_stride;
    a.vec[0] = vec_ok(g.k, g.k_row_stride, g.k_head_stride, g.type, 32);
    a.vec[1] = vec_ok(g.v, g.v_row_stride, g.v_head_stride, g.type, 32);
    a.status = status;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = g.type == MOSSGPU_F32   ? launch_read<float>(a, st)
                          : g.type == MOSSGPU_F16 ? launch_read<__half>(a, st)
                                                  : launch_read<__nv_bfloat16>(a, st);
    return e == cudaSuccess ? 0 : op_errorf("%s launch: %s", who, cudaGetErrorString(e));
}

size_t mossgpu_attention_kv8_workspace_bytes(const mossgpu_kv8_cache *cache, int q_heads, int rows) {
    if (!cache || q_heads <= 0 || rows <= 0 || cache->kv_heads < 1 || q_heads % cache->kv_heads ||
        (cache->head_dim != 64 && cache->head_dim != 128))
        return 0;
    return workspace_of(cache->head_dim, cache->kv_heads, int64_t(rows) * (q_heads / cache->kv_heads));
}

int mossgpu_attention_kv8(const mossgpu_kv8_cache *cache, const mossgpu_seq_batch *seqs, const mossgpu_attention_kv8_args *args,
                          void *cuda_stream) {
    const char *who = "attention_kv8";
    if (check_cache(cache, who) != 0) return 1;
    const int batch = check_seqs(seqs, who);
    if (batch > 0) return 1;
    if (!args) return op_errorf("%s: args is NULL", who);
    const mossgpu_attention_kv8_args &g = *args;
    if (!is_type(g.type)) return op_errorf("%s: type %d is no element type", who, g.type);
    if (g.q_heads < 1 || g.q_heads % cache->kv_heads)
        return op_errorf("%s: q_heads = %d must be a multiple of kv_heads = %d", who, g.q_heads, cache->kv_heads);
    if (!std::isfinite(g.scale)) return op_errorf("%s: scale is not finite", who);
    if (g.mask ? g.mask_words < 1 || g.mask_words > (1 << 20) : g.mask_words != 0)
        return op_errorf("%s: mask_words = %d does not fit the mask", who, g.mask_words);
    if (batch < 0) return 0;
    if (!g.q || !g.out || !g.workspace) return op_errorf("%s: a required pointer is NULL", who);
    if (!aligned(g.q, type_size(g.type)) || !aligned(g.out, type_size(g.type)) || !aligned(g.mask, 4))
        return op_errorf("%s: a pointer is not aligned to its type", who);
    if (!aligned(g.workspace, 16)) return op_errorf("%s: workspace must be 16-byte aligned", who);
    if (g.workspace_bytes < mossgpu_attention_kv8_workspace_bytes(cache, g.q_heads, seqs->rows))
        return op_errorf("%s: workspace too small (need mossgpu_attention_kv8_workspace_bytes)", who);
    if (!distinct(seqs->rows, g.q_heads, cache->head_dim, g.out_row_stride, g.out_head_stride))
        return op_errorf("%s: the strides of out make its heads overlap", who);
    if (g.q == g.out) return op_errorf("%s: out must not be q", who);
    const int group = g.q_heads / cache->kv_heads;
    const AttnForm f = attn_form(*cache, g.type, seqs->rows, seqs->n_seqs, group);
    const int64_t jobs = int64_t(seqs->rows) * g.q_heads;
    if (jobs > (int64_t(1) << 33)) return op_errorf("%s: rows * q_heads is above 2^33", who);
    if (int64_t(seqs->rows) * (g.q_heads / cache->kv_heads) > (1 << 30)) return op_errorf("%s: rows times heads of a group are above 2^30", who);
    // the plan counts tiles in 32 bits
    const int64_t blocks = int64_t(seqs->rows) * group / f.tile_rows + seqs->n_seqs;
    if (blocks * (cache->pages_per_slot / 2 + 1) >= int64_t(kKv8MaxTiles))
        return op_errorf("%s: rows times positions of the page table are above 2^31 tiles: split the call", who);
    int dev = -1, *status = nullptr;
    if (op_device(&dev, &status, who) != 0) return 1;
    AttnKv8 p{};
    p.cache = *cache;
    p.seqs = *seqs;
    p.a = g;
    p.group = group;
    p.runs = std::max(1, f.runs / cache->kv_heads);
    p.tile_rows = f.tile_rows;
    p.part_rows = int(std::min<int64_t>(f.tile_rows, int64_t(seqs->rows) * group));
    const int64_t units = (int64_t(seqs->rows) * group / f.tile_rows + seqs->n_seqs) * cache->kv_heads;
    p.vec_q = vec_ok(g.q, g.q_row_stride, g.q_head_stride, g.type, 16);
    p.vec_out = vec_ok(g.out, g.out_row_stride, g.out_head_stride, g.type, 16);
    p.plan = static_cast<uint32_t *>(g.workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(g.workspace) + plan_bytes());
    p.status = status;
    cudaError_t e = cudaFuncSetAttribute(f.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         f.ring + int(sizeof(uint32_t)) * (kAk8MaxSeqs + 1));
    if (e != cudaSuccess) return op_errorf("%s: cudaFuncSetAttribute: %s", who, cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(f.runs ? unsigned(kNumSMs * f.ctas) : unsigned(units));
    cfg.blockDim = dim3(unsigned(f.warps) * 32);
    cfg.dynamicSmemBytes = size_t(f.ring) + sizeof(uint32_t) * (seqs->n_seqs + 1);
    cfg.stream = static_cast<cudaStream_t>(cuda_stream);
    e = cudaLaunchKernelEx(&cfg, f.kernel, p);
    if (e != cudaSuccess) return op_errorf("%s launch: %s", who, cudaGetErrorString(e));
    if (f.runs == 0) return 0;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    // Few (row, head) pairs mean long units in many parts: a CTA each then (one stream of 4000 positions: the
    // join alone 66 us with a warp each), a warp each otherwise.
    const bool wide = jobs <= kNumSMs * 8;
    cfg.gridDim = dim3(unsigned(wide ? jobs : (jobs + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const auto join = cache->head_dim == 64 ? (wide ? k_attn_kv8_join<64, 8> : k_attn_kv8_join<64, 1>)
                                            : (wide ? k_attn_kv8_join<128, 8> : k_attn_kv8_join<128, 1>);
    e = cudaLaunchKernelEx(&cfg, join, p);
    return e == cudaSuccess ? 0 : op_errorf("%s join launch: %s", who, cudaGetErrorString(e));
}

}  // extern "C"
