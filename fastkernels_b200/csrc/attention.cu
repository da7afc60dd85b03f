// Attention of new tokens over a paged cache: entry point, the kernel for any type, size and alignment, and the joining of
// partial results.
//
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale * q . k_j over the visible j, m the running maximum; all
// sums and statistics in fp32.  Pieces (m, l, acc) of one row over disjoint keys join as
// m = max m_i, l = sum 2^(m_i - m) l_i, acc = sum 2^(m_i - m) acc_i.

#include <cfloat>
#include <cmath>

#include "attention.cuh"

namespace fk {

constexpr int kAnyWarps = 4;

// One warp per (row, query head, piece of the key axis).
template <typename T, typename TC, bool WIDE>
__global__ void __launch_bounds__(32 * kAnyWarps) attention_any_kernel(const __grid_constant__ AttnParams p) {
    __shared__ float q_rows[kAnyWarps][FK_MAX_HEAD_DIM + 8];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.head_dim;
    const int64_t item = (int64_t)blockIdx.x * kAnyWarps + warp;
    if (item >= (int64_t)p.rows * p.q_heads * p.splits) return;
    const int64_t rh = item / p.splits;
    const int split = (int)(item - rh * p.splits);
    const int row = (int)(rh / p.q_heads), qh = (int)(rh - (int64_t)row * p.q_heads);
    const RowPlace at = place_of_row(p.starts, p.c.lengths, p.c.seqs, p.rows, row);
    T* out = reinterpret_cast<T*>(p.out) + row * p.os[0] + qh * p.os[1];
    RowSums r;
    if (at.seq < 0) {
        if (split == 0 && p.zero_rest)
            for (int d = lane; d < D; d += 32) store_elem(out + d, 0.f);
        if (p.splits == 1) return;
        r.m = -INFINITY;
        r.l = -1.f;                              // marks a row that is left alone
    } else {
        float* q = q_rows[warp];
        const T* query = reinterpret_cast<const T*>(p.query) + row * p.qs[0] + qh * p.qs[1];
        for (int d = lane; d < D + 8; d += 32) q[d] = d < D ? load_elem(query + d) * p.scale_log2 : 0.f;
        __syncwarp();
        warp_row<TC, WIDE>(p, [q](int d) { return q[d]; }, at.seq, qh / p.group, at.pos, split, p.splits, r);
    }
    if (p.splits == 1) {
        const float inv = r.l > 0.f || r.l != r.l ? 1.f / r.l : 0.f;
#pragma unroll
        for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
            if (c * 32 + lane < D) store_elem(out + c * 32 + lane, r.l == 0.f ? 0.f : r.acc[c] * inv);
        return;
    }
    float* part = p.part + item * (D + 2);
    if (lane == 0) { part[0] = r.m; part[1] = r.l; }
    if (r.l > 0.f || r.l != r.l)
#pragma unroll
        for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
            if (c * 32 + lane < D) part[2 + c * 32 + lane] = r.acc[c];
}

template <typename T>
__global__ void __launch_bounds__(32 * kAnyWarps) attention_any_join_kernel(const __grid_constant__ AttnParams p) {
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.head_dim;
    const int64_t rh = (int64_t)blockIdx.x * kAnyWarps + warp;
    if (rh >= (int64_t)p.rows * p.q_heads) return;
    const int row = (int)(rh / p.q_heads), qh = (int)(rh - (int64_t)row * p.q_heads);
    const float* part = p.part + rh * p.splits * (D + 2);
    if (part[1] == -1.f) return;
    float m = -INFINITY, l = 0.f, acc[FK_MAX_HEAD_DIM / 32] = {};
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, part[(int64_t)s * (D + 2)]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int s = 0; s < p.splits; ++s) {
        const float* one = part + (int64_t)s * (D + 2);
        if (one[1] == 0.f) continue;
        const float w = exp2f(one[0] - base);
        l = fmaf(w, one[1], l);
#pragma unroll
        for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
            if (c * 32 + lane < D) acc[c] = fmaf(w, one[2 + c * 32 + lane], acc[c]);
    }
    T* out = reinterpret_cast<T*>(p.out) + row * p.os[0] + qh * p.os[1];
#pragma unroll
    for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
        if (c * 32 + lane < D) store_elem(out + c * 32 + lane, l == 0.f ? 0.f : acc[c] / l);
}

static int check_attention(const fk_attention_call* a) {
    if (a == nullptr) return FK_ERR_ARG;
    const int st = check_cache(a->cache);
    if (st != FK_OK) return st;
    if (a->dtype != FK_F32 && a->dtype != FK_BF16 && a->dtype != FK_F16) return FK_ERR_UNSUPPORTED;
    if (a->cache.dtype != FK_E4M3 && a->cache.dtype != a->dtype) return FK_ERR_UNSUPPORTED;
    if (a->rows < 0 || a->q_heads < 1 || a->q_heads % a->cache.kv_heads != 0) return FK_ERR_ARG;
    if ((int64_t)a->rows * a->q_heads > INT32_MAX || a->window < 0 || a->sinks < 0 || a->max_query < 0) return FK_ERR_ARG;
    if (a->rows > 0 && (!a->query || !a->out)) return FK_ERR_ARG;
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return FK_ERR_ARG;      // NaN or infinite
    return FK_OK;
}

// Pieces of the key axis: enough warps for the whole chip (16 per SM) where there are few rows, none shorter than 64 keys.
static int any_splits(const fk_attention_call& a) {
    const int64_t rows = (int64_t)a.rows * a.q_heads;
    const int64_t longest = (int64_t)a.cache.max_pages * a.cache.page_size;
    int64_t want = (148 * 16 + rows - 1) / rows;
    if (want > (longest + 63) / 64) want = (longest + 63) / 64;
    if (want > 64) want = 64;
    return want < 1 ? 1 : (int)want;
}

template <typename T, typename TC>
static int launch_any(const AttnParams& p, bool wide, cudaStream_t stream) {
    const int64_t items = (int64_t)p.rows * p.q_heads * p.splits;
    auto kern = wide ? attention_any_kernel<T, TC, true> : attention_any_kernel<T, TC, false>;
    FK_CUDA_OK(launch_pdl(kern, dim3((unsigned)((items + kAnyWarps - 1) / kAnyWarps)), dim3(32 * kAnyWarps), 0, stream, p), "attention launch");
    FK_LAUNCH_OK("attention launch");
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.rows * p.q_heads;
        FK_CUDA_OK(launch_pdl(attention_any_join_kernel<T>, dim3((unsigned)((rows + kAnyWarps - 1) / kAnyWarps)), dim3(32 * kAnyWarps), 0, stream, p),
                   "attention join launch");
        FK_LAUNCH_OK("attention join launch");
    }
    return FK_OK;
}

static AttnParams attn_params(const fk_attention_call& a) {
    AttnParams p{};
    p.c = a.cache;
    p.query = a.query; p.out = a.out; p.starts = a.starts;
    for (int i = 0; i < 2; ++i) { p.qs[i] = a.query_stride[i]; p.os[i] = a.out_stride[i]; }
    p.rows = a.rows; p.q_heads = a.q_heads; p.group = a.q_heads / a.cache.kv_heads;
    p.window = a.window; p.sinks = a.window > 0 ? a.sinks : 0; p.zero_rest = a.zero_rest;
    p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
    if (fabsf(p.scale_log2) < FLT_MIN) p.scale_log2 = FLT_MIN;
    p.part = reinterpret_cast<float*>(a.workspace);
    return p;
}

enum class Path { any, few, tile };

// Few rows per key/value head (up to 16, 8 at 256 dimensions: decode and short continuations) are a stream of the cache; more, and head sizes that
// the stream has no form for, go to the tensor cores; fp32, head sizes off a multiple of 8 and rows off 16-byte boundaries take
// the shape-agnostic kernel.
static Path path_of(const fk_attention_call& a, const AttnParams& p) {
    if (a.flags & FK_FLAG_FORCE_GENERIC) return Path::any;
    const int most = a.starts == nullptr ? 1 : a.max_query;
    if (attention_few_supported(p, a.dtype, most)) return Path::few;
    if (attention_tile_supported(p, a.dtype)) return Path::tile;
    return Path::any;
}

static size_t workspace_need(const fk_attention_call& a, const AttnParams& p, Path path) {
    size_t need = 0;
    if (path == Path::few) {
        attention_few(p, a.dtype, a.starts == nullptr ? 1 : a.max_query, &need, nullptr);
        return need;
    }
    if (path == Path::tile) {
        attention_tile(p, a.dtype, &need, nullptr);
        return need;
    }
    const int splits = any_splits(a);
    return splits > 1 ? (size_t)a.rows * a.q_heads * splits * (a.cache.head_dim + 2) * sizeof(float) : 0;
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fk_paged_attention_workspace_bytes(const fk_attention_call* a) {
    if (check_attention(a) != FK_OK || a->rows == 0) return 0;
    const AttnParams p = attn_params(*a);
    return workspace_need(*a, p, path_of(*a, p));
}

int fk_paged_attention(const fk_attention_call* a, void* stream) {
    const int st = check_attention(a);
    if (st != FK_OK) return st;
    if (a->rows == 0 || (a->cache.seqs == 0 && !a->zero_rest)) return FK_OK;
    AttnParams p = attn_params(*a);
    const Path path = path_of(*a, p);
    const size_t need = workspace_need(*a, p, path);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 15))) return FK_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    if (path == Path::few) return attention_few(p, a->dtype, a->starts == nullptr ? 1 : a->max_query, nullptr, s);
    if (path == Path::tile) return attention_tile(p, a->dtype, nullptr, s);
    p.splits = any_splits(*a);
    const int cb = dtype_bytes(a->cache.dtype);
    const bool wide = a->cache.head_dim % 8 == 0 && groups_aligned(a->cache.key, a->cache.key_stride, 3, cb, cb == 1 ? 8 : 16);
    if (a->cache.dtype == FK_E4M3) {
        if (a->dtype == FK_BF16) return launch_any<__nv_bfloat16, __nv_fp8_e4m3>(p, wide, s);
        if (a->dtype == FK_F16) return launch_any<__half, __nv_fp8_e4m3>(p, wide, s);
        return launch_any<float, __nv_fp8_e4m3>(p, wide, s);
    }
    if (a->dtype == FK_BF16) return launch_any<__nv_bfloat16, __nv_bfloat16>(p, wide, s);
    if (a->dtype == FK_F16) return launch_any<__half, __half>(p, wide, s);
    return launch_any<float, float>(p, wide, s);
}

}
