// Paged key/value cache: new tokens written (as they are, or as e4m3 codes with a scale per row) and read back.
//
// A row is one token's head_dim elements of one head.  Eight elements per lane, ceil(head_dim / 8) lanes per row rounded
// up to a power of two, so a 256-element row is a warp and a 128-element row half of one.  Both kernels are streams of
// bytes; the row's maximum is one group-wide shuffle reduction.

#include "kv_cache.cuh"

namespace fk {

int dtype_bytes(int dtype) { return dtype == FK_F32 ? 4 : dtype == FK_E4M3 ? 1 : 2; }

int check_cache(const fk_kv_cache& c) {
    if (c.pages < 1 || c.kv_heads < 1 || c.page_size < 1 || c.head_dim < 1 || c.head_dim > FK_MAX_HEAD_DIM) return FK_ERR_ARG;
    if (c.seqs < 0 || c.max_pages < 0 || c.table_stride < 0) return FK_ERR_ARG;
    if ((int64_t)c.max_pages * c.page_size > INT32_MAX) return FK_ERR_ARG;
    if (c.dtype < FK_F32 || c.dtype > FK_E4M3) return FK_ERR_UNSUPPORTED;
    if (!c.key || !c.value) return FK_ERR_ARG;
    if (c.seqs > 0 && (!c.lengths || (c.max_pages > 0 && !c.page_table))) return FK_ERR_ARG;
    if (c.dtype == FK_E4M3 && (!c.key_scale || !c.value_scale)) return FK_ERR_ARG;
    return FK_OK;
}

bool groups_aligned(const void* base, const int64_t* stride, int n, int bytes, int align) {
    if (reinterpret_cast<uintptr_t>(base) % align) return false;
    for (int i = 0; i < n; ++i)
        if ((stride[i] * bytes) % align) return false;
    return true;
}

// NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct KvParams {
    fk_kv_cache c;
    fk_kv_rows r;
    int group_log2;            // lanes per row, as a power of two
};

template <typename T, typename TC, bool WIDE>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ KvParams p) {
    pdl_trigger();
    pdl_wait();
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> p.group_log2;
    const int lane = threadIdx.x & ((1 << p.group_log2) - 1);
    const int per_token = 2 * p.c.kv_heads;
    if (item >= (int64_t)p.r.rows * per_token) return;          // whole groups leave together
    const int row = (int)(item / per_token), rest = (int)(item - (int64_t)row * per_token);
    const bool is_value = rest >= p.c.kv_heads;
    const int head = is_value ? rest - p.c.kv_heads : rest;
    const int d0 = lane * 8, n = min(8, p.c.head_dim - d0);
    const int64_t* from = is_value ? p.r.value_stride : p.r.key_stride;
    float v[8] = {};
    if (n > 0) load8<WIDE>(reinterpret_cast<const T*>(is_value ? p.r.value : p.r.key) + row * from[0] + head * from[1] + d0, n, v);
    const RowPlace at = place_of_row(p.r.starts, p.c.lengths, p.c.seqs, p.r.rows, row);
    int in_page = 0;
    const int page = at.seq < 0 ? -1 : page_of(p.c, at.seq, at.pos, in_page);
    if (sizeof(TC) == 1) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(v[i]));
        const unsigned mask = p.group_log2 == 5 ? kFull : ((1u << (1 << p.group_log2)) - 1u) << ((threadIdx.x & 31) & ~((1 << p.group_log2) - 1));
        for (int o = 1 << p.group_log2 >> 1; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(mask, most, o));
        most = max_nan(most, 0x1p-100f);
        // x * 448 / most with one rounding, so that quotients half way between two codes stay there; both factors carry
        // 2^-9 so that the product cannot overflow
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (v[i] * 0.875f) / (most * 0x1p-9f);
        if (lane == 0 && page >= 0) {
            const int64_t* to = is_value ? p.c.value_scale_stride : p.c.key_scale_stride;
            float* s = is_value ? p.c.value_scale : p.c.key_scale;
            s[page * to[0] + head * to[1] + in_page * to[2]] = most / 448.0f;
        }
    }
    if (page < 0 || n <= 0) return;
    const int64_t* to = is_value ? p.c.value_stride : p.c.key_stride;
    store8<WIDE>(reinterpret_cast<TC*>(is_value ? p.c.value : p.c.key) + page * to[0] + head * to[1] + in_page * to[2] + d0, n, v);
}

template <typename T, typename TC, bool WIDE>
__global__ void __launch_bounds__(256) kv_gather_kernel(const __grid_constant__ KvParams p) {
    pdl_trigger();
    pdl_wait();
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> p.group_log2;
    const int lane = threadIdx.x & ((1 << p.group_log2) - 1);
    const int per_token = 2 * p.c.kv_heads;
    if (item >= (int64_t)p.r.rows * per_token) return;
    const int row = (int)(item / per_token), rest = (int)(item - (int64_t)row * per_token);
    const bool is_value = rest >= p.c.kv_heads;
    const int head = is_value ? rest - p.c.kv_heads : rest;
    const int d0 = lane * 8, n = min(8, p.c.head_dim - d0);
    const RowPlace at = place_of_row(p.r.starts, p.c.lengths, p.c.seqs, p.r.rows, row);
    if (n <= 0 || (at.seq < 0 && !p.r.zero_rest)) return;
    int in_page = 0;
    const int page = at.seq < 0 ? -1 : page_of(p.c, at.seq, at.pos, in_page);
    float v[8] = {};
    if (page >= 0) {
        const int64_t* from = is_value ? p.c.value_stride : p.c.key_stride;
        load8<WIDE>(reinterpret_cast<const TC*>(is_value ? p.c.value : p.c.key) + page * from[0] + head * from[1] + in_page * from[2] + d0, n, v);
        if (sizeof(TC) == 1) {
            const int64_t* sf = is_value ? p.c.value_scale_stride : p.c.key_scale_stride;
            const float s = (is_value ? p.c.value_scale : p.c.key_scale)[page * sf[0] + head * sf[1] + in_page * sf[2]];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= s;
        }
    }
    const int64_t* to = is_value ? p.r.value_stride : p.r.key_stride;
    store8<WIDE>(reinterpret_cast<T*>(is_value ? p.r.value : p.r.key) + row * to[0] + head * to[1] + d0, n, v);
}

static int check_rows(const fk_kv_cache& c, const fk_kv_rows& r) {
    if (r.rows < 0) return FK_ERR_ARG;
    if (r.dtype != FK_F32 && r.dtype != FK_BF16 && r.dtype != FK_F16) return FK_ERR_UNSUPPORTED;
    if (c.dtype != FK_E4M3 && c.dtype != r.dtype) return FK_ERR_UNSUPPORTED;
    if (r.rows > 0 && (!r.key || !r.value)) return FK_ERR_ARG;
    return FK_OK;
}

template <bool APPEND, typename T, typename TC>
static int launch_rows(const KvParams& p, bool wide, cudaStream_t stream) {
    const int64_t threads = ((int64_t)p.r.rows * 2 * p.c.kv_heads) << p.group_log2;
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > INT32_MAX) return FK_ERR_ARG;
    auto kern = APPEND ? (wide ? kv_append_kernel<T, TC, true> : kv_append_kernel<T, TC, false>)
                       : (wide ? kv_gather_kernel<T, TC, true> : kv_gather_kernel<T, TC, false>);
    FK_CUDA_OK(launch_pdl(kern, dim3((unsigned)blocks), dim3(256), 0, stream, p), APPEND ? "kv append launch" : "kv gather launch");
    FK_LAUNCH_OK(APPEND ? "kv append launch" : "kv gather launch");
    return FK_OK;
}

template <bool APPEND>
static int kv_rows(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) {
    if (cache == nullptr || rows == nullptr) return FK_ERR_ARG;
    int st = check_cache(*cache);
    if (st != FK_OK) return st;
    st = check_rows(*cache, *rows);
    if (st != FK_OK) return st;
    if (rows->rows == 0 || (cache->seqs == 0 && (APPEND || !rows->zero_rest))) return FK_OK;
    KvParams p{*cache, *rows, 0};
    while ((8 << p.group_log2) < cache->head_dim) ++p.group_log2;
    const int rb = dtype_bytes(rows->dtype), cb = dtype_bytes(cache->dtype);
    const bool wide = cache->head_dim % 8 == 0 && groups_aligned(rows->key, rows->key_stride, 2, rb, 16) &&
                      groups_aligned(rows->value, rows->value_stride, 2, rb, 16) &&
                      groups_aligned(cache->key, cache->key_stride, 3, cb, cb == 1 ? 8 : 16) &&
                      groups_aligned(cache->value, cache->value_stride, 3, cb, cb == 1 ? 8 : 16);
    cudaStream_t s = (cudaStream_t)stream;
    if (cache->dtype == FK_E4M3) {
        if (rows->dtype == FK_BF16) return launch_rows<APPEND, __nv_bfloat16, __nv_fp8_e4m3>(p, wide, s);
        if (rows->dtype == FK_F16) return launch_rows<APPEND, __half, __nv_fp8_e4m3>(p, wide, s);
        return launch_rows<APPEND, float, __nv_fp8_e4m3>(p, wide, s);
    }
    if (rows->dtype == FK_BF16) return launch_rows<APPEND, __nv_bfloat16, __nv_bfloat16>(p, wide, s);
    if (rows->dtype == FK_F16) return launch_rows<APPEND, __half, __half>(p, wide, s);
    return launch_rows<APPEND, float, float>(p, wide, s);
}

}  // namespace fk

extern "C" {

int fk_kv_append(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) { return fk::kv_rows<true>(cache, rows, stream); }
int fk_kv_gather(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) { return fk::kv_rows<false>(cache, rows, stream); }

}
