// Attention of new tokens over a paged cache: entry point, the kernel for any type, size and alignment, and the joining of
// partial results.
//
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale * q . k_j over the visible j, m the running maximum; all
// sums and statistics in fp32.  Pieces (m, l, acc) of one row over disjoint keys join as
// m = max m_i, l = sum 2^(m_i - m) l_i, acc = sum 2^(m_i - m) acc_i.

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.cuh"
#include "kernels.cuh"

namespace fk {

constexpr int kAnyWarps = 4;
constexpr int kAnyKeys = 32;           // of a tile
constexpr int kAnyHeads = 4;           // query heads per warp

// dimensions of a row in shared memory: a multiple of 8, and 4 more so that 32 rows' 16-byte pieces lie in different banks
__host__ __device__ constexpr int any_pitch(int dim) { return (dim + 7) / 8 * 8 + 4; }
__host__ __device__ inline int any_smem(int dim, int heads) { return (2 * kAnyKeys * any_pitch(dim) + heads * any_pitch(dim)) * (int)sizeof(float); }

// Any type, size and alignment, on the CUDA cores in fp32.  Block = (token, key/value head, up to 16 of its query heads, piece of the key
// axis).  32 keys and values at a time are brought into shared memory as fp32 by coalesced loads, once for all heads; then a warp per
// head takes one key per lane for the scores (no reduction per key) and one column per lane for the values.  What bounds it is the
// shared-memory reads of the products (one per four multiply-adds in the scores, one per multiply-add in the values); a row per warp
// straight from L2, without the tile, took 55 us where this takes 24 (61 tokens at up to 700, 6 heads of 80 in fp32).
// NC: groups of 32 columns, at least head_dim / 32.
template <typename T, typename TC, bool WIDE, int NC>
__global__ void __launch_bounds__(32 * kAnyWarps) attention_any_kernel(const __grid_constant__ AttnParams p) {
    extern __shared__ __align__(16) float any_tile[];
    __shared__ unsigned there;
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.head_dim, pitch = any_pitch(D), Dp = pitch - 4;
    const int head_blocks = (p.group + kAnyWarps * kAnyHeads - 1) / (kAnyWarps * kAnyHeads);
    int64_t at_block = blockIdx.x;
    const int split = (int)(at_block % p.splits);
    at_block /= p.splits;
    const int head_block = (int)(at_block % head_blocks);
    at_block /= head_blocks;
    const int kv_head = (int)(at_block % p.c.kv_heads), row = (int)(at_block / p.c.kv_heads);
    const int head0 = kv_head * p.group + head_block * kAnyWarps * kAnyHeads, heads = min(kAnyWarps * kAnyHeads, p.group - head_block * kAnyWarps * kAnyHeads);
    float* keys = any_tile;
    float* values = keys + kAnyKeys * pitch;
    float* queries = values + kAnyKeys * pitch;
    const RowPlace at = place_of_row(p.starts, p.c.lengths, p.c.seqs, p.rows, row);
    float m[kAnyHeads], l[kAnyHeads], acc[kAnyHeads][NC];
#pragma unroll
    for (int i = 0; i < kAnyHeads; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = 0.f;
    }
    if (at.seq >= 0) {
        const T* query = reinterpret_cast<const T*>(p.query) + row * p.qs[0] + head0 * p.qs[1];
        for (int i = threadIdx.x; i < heads * Dp; i += blockDim.x) {
            const int a = i / Dp, d = i - a * Dp;
            queries[a * pitch + d] = d < D ? load_elem(query + a * p.qs[1] + d) * p.scale_log2 : 0.f;
        }
        const int end = min(at.pos + 1, p.c.max_pages * p.c.page_size);      // positions that the table does not hold are not visible
        const int lo = window_start(p, at.pos), n_sinks = max(0, min(p.sinks, min(lo, end)));
        const int count = n_sinks + max(0, end - lo);
        const int pieces = Dp / 8;
        for (int64_t k0 = (int64_t)split * kAnyKeys; k0 < count; k0 += (int64_t)p.splits * kAnyKeys) {
            __syncthreads();                         // the last tile has been read
            // every warp looks all 32 keys up, one per lane
            const int64_t k = k0 + lane;
            int in_page = 0, page = -1;
            if (k < count) page = page_of(p.c, at.seq, (int)(k < n_sinks ? k : lo + k - n_sinks), in_page);
            const int64_t koff = page < 0 ? -1 : row_offset(p.c.key_stride, page, kv_head, in_page), voff = page < 0 ? -1 : row_offset(p.c.value_stride, page, kv_head, in_page);
            float kscale = 1.f, vscale = 1.f;
            if (sizeof(TC) == 1 && page >= 0) {
                kscale = p.c.key_scale[row_offset(p.c.key_scale_stride, page, kv_head, in_page)];
                vscale = p.c.value_scale[row_offset(p.c.value_scale_stride, page, kv_head, in_page)];
            }
            if (warp == 0) {
                const unsigned bits = __ballot_sync(kFull, page >= 0);
                if (lane == 0) there = bits;
            }
            // 8 rows per warp: lanes over their pieces of eight elements
#pragma unroll 2
            for (int i0 = 0; i0 < 8 * pieces; i0 += 32) {
                const int i = i0 + lane, r = warp * 8 + min(i / pieces, 7), d = (i - (i / pieces) * pieces) * 8;
                const int64_t ko = __shfl_sync(kFull, koff, r), vo = __shfl_sync(kFull, voff, r);
                const float ks = __shfl_sync(kFull, kscale, r), vs = __shfl_sync(kFull, vscale, r);
                if (i >= 8 * pieces) continue;
                float a[8] = {}, b[8] = {};
                if (ko >= 0) {
                    load8<WIDE>(reinterpret_cast<const TC*>(p.c.key) + ko + d, D - d, a);
                    load8<WIDE>(reinterpret_cast<const TC*>(p.c.value) + vo + d, D - d, b);
                }
                if (sizeof(TC) == 1) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        a[e] = ko >= 0 ? a[e] * ks : 0.f;
                        b[e] = ko >= 0 ? b[e] * vs : 0.f;
                    }
                }
                store8<true>(keys + r * pitch + d, 8, a);
                store8<true>(values + r * pitch + d, 8, b);
            }
            __syncthreads();
            const unsigned seen = there;
            if (seen == 0) continue;
#pragma unroll
            for (int i = 0; i < kAnyHeads; ++i) {
                const int a = warp + i * kAnyWarps;
                if (a >= heads) continue;
                const float4* q = reinterpret_cast<const float4*>(queries + a * pitch);
                const float4* kr = reinterpret_cast<const float4*>(keys + lane * pitch);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int d = 0; d < Dp / 4; ++d) {
                    const float4 x = q[d], y = kr[d];
                    sum[0] = fmaf(x.x, y.x, sum[0]); sum[1] = fmaf(x.y, y.y, sum[1]);
                    sum[2] = fmaf(x.z, y.z, sum[2]); sum[3] = fmaf(x.w, y.w, sum[3]);
                }
                const bool mine = (seen >> lane) & 1u;
                const float s = mine ? (sum[0] + sum[1]) + (sum[2] + sum[3]) : -INFINITY;
                const float m_new = fmaxf(m[i], warp_max(s));
                const float base = m_new == -INFINITY ? 0.f : m_new;        // nothing but scores of -infinity so far
                const float alpha = exp2f(m[i] - base), w = mine ? exp2f(s - base) : 0.f;
                m[i] = m_new;
                l[i] = l[i] * alpha + warp_sum(w);
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[i][c] *= alpha;
#pragma unroll 4
                for (int r = 0; r < kAnyKeys; ++r) {
                    const float wr = __shfl_sync(kFull, w, r);
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        acc[i][c] = fmaf(wr, values[r * pitch + min(c * 32 + lane, Dp - 1)], acc[i][c]);
                }
            }
        }
    }
    if (at.seq < 0 && !p.zero_rest && p.splits == 1) return;
#pragma unroll
    for (int i = 0; i < kAnyHeads; ++i) {
        const int a = warp + i * kAnyWarps;
        if (a >= heads) continue;
        const int64_t rh = (int64_t)row * p.q_heads + head0 + a;
        if (p.splits == 1) {
            T* out = reinterpret_cast<T*>(p.out) + row * p.os[0] + (head0 + a) * p.os[1];
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (c * 32 + lane < D) store_elem(out + c * 32 + lane, l[i] == 0.f ? 0.f : acc[i][c] / l[i]);
            continue;
        }
        float* part = p.part + (rh * p.splits + split) * (D + 2);
        if (lane == 0) {
            part[0] = m[i];
            part[1] = at.seq < 0 && !p.zero_rest ? -1.f : l[i];          // -1: a row that is left alone
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (c * 32 + lane < D) part[2 + c * 32 + lane] = acc[i][c];
    }
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
    // a lane per piece (64 at most) for the statistics, then a lane per column for the sums
    float pm[2], pl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = lane + 32 * i;
        pm[i] = s < p.splits ? part[(int64_t)s * (D + 2)] : -INFINITY;
        pl[i] = s < p.splits ? part[(int64_t)s * (D + 2) + 1] : 0.f;
    }
    if (__shfl_sync(kFull, pl[0], 0) == -1.f) return;
    const float m = warp_max(fmaxf(pm[0], pm[1])), base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 2; ++i) pm[i] = exp2f(pm[i] - base);
    const float l = warp_sum(pm[0] * pl[0] + pm[1] * pl[1]);
    float acc[FK_MAX_HEAD_DIM / 32] = {};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = __shfl_sync(kFull, s < 32 ? pm[0] : pm[1], s & 31);
        const float* one = part + (int64_t)s * (D + 2) + 2;
#pragma unroll
        for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
            if (c * 32 + lane < D) acc[c] = fmaf(w, one[c * 32 + lane], acc[c]);
    }
    T* out = reinterpret_cast<T*>(p.out) + row * p.os[0] + qh * p.os[1];
#pragma unroll
    for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
        if (c * 32 + lane < D) store_elem(out + c * 32 + lane, l == 0.f ? 0.f : acc[c] / l);
}

constexpr double kLog2E = 1.4426950408889634;

static int check_attention(const fk_attention_call* a) {
    if (a == nullptr) return FK_ERR_ARG;
    const int st = check_cache(a->cache);
    if (st != FK_OK) return st;
    if (a->dtype != FK_F32 && a->dtype != FK_BF16 && a->dtype != FK_F16) return FK_ERR_UNSUPPORTED;
    if (a->cache.dtype != FK_E4M3 && a->cache.dtype != a->dtype) return FK_ERR_UNSUPPORTED;
    if (a->rows < 0 || a->q_heads < 1 || a->q_heads % a->cache.kv_heads != 0) return FK_ERR_ARG;
    if ((int64_t)a->rows * a->q_heads > INT32_MAX || a->window < 0 || a->sinks < 0 || a->max_query < 0) return FK_ERR_ARG;
    if (a->rows > 0 && (!a->query || !a->out)) return FK_ERR_ARG;
    if (!(fabs((double)a->scale) * kLog2E <= FLT_MAX)) return FK_ERR_ARG;      // NaN, infinite, or infinite as a power of two
    return FK_OK;
}

static int64_t any_blocks(const fk_attention_call& a) {
    const int group = a.q_heads / a.cache.kv_heads;
    return (int64_t)a.rows * a.cache.kv_heads * ((group + kAnyWarps * kAnyHeads - 1) / (kAnyWarps * kAnyHeads));
}

// Pieces of the key axis: enough blocks for the whole chip (8 per SM) where there are few rows, none shorter than 64 keys.
static int any_splits(const fk_attention_call& a) {
    const int64_t blocks = any_blocks(a), longest = (int64_t)a.cache.max_pages * a.cache.page_size;
    int64_t want = ((int64_t)sm_count() * 8 + blocks - 1) / blocks;
    if (want > (longest + 63) / 64) want = (longest + 63) / 64;
    if (want > 64) want = 64;
    return want < 1 ? 1 : (int)want;
}

template <typename T, typename TC>
static int launch_any(const AttnParams& p, int64_t blocks, bool wide, cudaStream_t stream) {
    const int columns = p.c.head_dim <= 64 ? 0 : p.c.head_dim <= 128 ? 1 : 2;
    auto pick = [&](auto few, auto some, auto all) { return columns == 0 ? few : columns == 1 ? some : all; };
    auto kern = wide ? pick(attention_any_kernel<T, TC, true, 2>, attention_any_kernel<T, TC, true, 4>, attention_any_kernel<T, TC, true, 8>)
                     : pick(attention_any_kernel<T, TC, false, 2>, attention_any_kernel<T, TC, false, 4>, attention_any_kernel<T, TC, false, 8>);
    const int heads = p.group < kAnyWarps * kAnyHeads ? p.group : kAnyWarps * kAnyHeads, smem = any_smem(p.c.head_dim, heads);
    static std::atomic<uint64_t> allowed[2][3];
    FK_CUDA_OK(allow_smem(kern, any_smem(FK_MAX_HEAD_DIM, kAnyWarps * kAnyHeads), allowed[wide][columns]), "attention attr");
    FK_CUDA_OK(launch_pdl(kern, dim3((unsigned)(blocks * p.splits)), dim3(32 * kAnyWarps), (size_t)smem, stream, p), "attention launch");
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
    p.scale_log2 = (float)((double)a.scale * kLog2E);
    if (fabsf(p.scale_log2) < FLT_MIN) p.scale_log2 = FLT_MIN;
    p.part = reinterpret_cast<float*>(a.workspace);
    p.wait_cycles = (uint32_t)std::min(wait_limit_cycles(), 1ll << 31);       // clocks are compared in 32 bits
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
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 31))) return FK_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    if (path == Path::few) return attention_few(p, a->dtype, a->starts == nullptr ? 1 : a->max_query, nullptr, s);
    if (path == Path::tile) return attention_tile(p, a->dtype, nullptr, s);
    p.splits = any_splits(*a);
    const int cb = dtype_bytes(a->cache.dtype);
    const bool wide = a->cache.head_dim % 8 == 0 && groups_aligned(a->cache.key, a->cache.key_stride, 3, cb, cb == 1 ? 8 : 16) &&
                      groups_aligned(a->cache.value, a->cache.value_stride, 3, cb, cb == 1 ? 8 : 16);
    if (a->cache.dtype == FK_E4M3) {
        if (a->dtype == FK_BF16) return launch_any<__nv_bfloat16, __nv_fp8_e4m3>(p, any_blocks(*a), wide, s);
        if (a->dtype == FK_F16) return launch_any<__half, __nv_fp8_e4m3>(p, any_blocks(*a), wide, s);
        return launch_any<float, __nv_fp8_e4m3>(p, any_blocks(*a), wide, s);
    }
    if (a->dtype == FK_BF16) return launch_any<__nv_bfloat16, __nv_bfloat16>(p, any_blocks(*a), wide, s);
    if (a->dtype == FK_F16) return launch_any<__half, __half>(p, any_blocks(*a), wide, s);
    return launch_any<float, float>(p, any_blocks(*a), wide, s);
}

}
