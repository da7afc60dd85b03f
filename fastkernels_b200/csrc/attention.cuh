// Paged attention: what its kernels share.
#pragma once

#include <atomic>

#include "kv_cache.cuh"

namespace fk {

struct AttnParams {
    fk_kv_cache c;
    const void* query;
    void* out;
    const int* starts;
    int64_t qs[2], os[2];      // row, head
    int rows, q_heads, group;  // group = query heads per key/value head
    int window, sinks, zero_rest;
    float scale_log2;          // scale * log2(e): scores are held as powers of two; never zero, so that masked scores stay -infinity
    int splits;                // pieces of the key axis (shape-agnostic kernel)
    float* part;               // partial results
    int tile_tokens;           // tokens of an item of the kernels that work on tiles of tokens
    uint32_t wait_cycles;      // limit of every wait for a barrier
};

// What a token at position p sees: [0, min(sinks, lo)) and [lo, p], lo = first position of its window.
__device__ __forceinline__ int window_start(const AttnParams& p, int pos) { return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0; }

__device__ __forceinline__ float load_elem(const float* p) { return *p; }
__device__ __forceinline__ float load_elem(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_elem(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_elem(const __nv_fp8_e4m3* p) { return (float)*p; }
__device__ __forceinline__ void store_elem(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_elem(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_elem(__half* p, float v) { *p = __float2half_rn(v); }

// Exponent by which a query row of largest magnitude `most` is brought to fp16.  Not below -126: 2^-it has to be a number, and a row of
// subnormal elements needs no more.
__device__ __forceinline__ int row_exponent(float most) { return most > 0.f && most < INFINITY ? max(ilogbf(most), -126) : 0; }

// The sums of one row over some keys, held by a warp: lane l has the elements l, l + 32, ... of acc.
struct RowSums {
    float m, l;
    float acc[FK_MAX_HEAD_DIM / 32];
};

// A row that is computed again (row_again): one warp, one query row (q(d) is element d times scale * log2 e, q(d >= head_dim) anything finite): groups first, first + step, ..
// of 32 of the visible keys.  One lane computes one key's score (no reduction per key); then the value rows are added one at
// a time, a lane per column.  Keys that are masked never enter any sum, whatever their rows hold.
template <typename TC, bool WIDE, typename Q>
__device__ __forceinline__ void warp_row(const AttnParams& p, const Q& q, int seq, int head, int pos, int first, int step, RowSums& r) {
    const int lane = threadIdx.x & 31, D = p.c.head_dim;
    const int end = min(pos + 1, p.c.max_pages * p.c.page_size);       // positions that the table does not hold are not visible
    const int lo = window_start(p, pos), n_sinks = max(0, min(p.sinks, min(lo, end)));
    const int count = n_sinks + max(0, end - lo);
    r.m = -INFINITY;
    r.l = 0.f;
#pragma unroll
    for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c) r.acc[c] = 0.f;
    const TC* keys = reinterpret_cast<const TC*>(p.c.key) + head * p.c.key_stride[1];
    const TC* values = reinterpret_cast<const TC*>(p.c.value) + head * p.c.value_stride[1];
    // where the key of this lane in the group at k0 is; looked up one group ahead of its use
    int next_page = -1, next_row = 0;
    auto look = [&](int64_t k0) {
        next_page = -1;
        const int64_t k = k0 + lane;
        if (k < count) next_page = page_of(p.c, seq, (int)(k < n_sinks ? k : lo + k - n_sinks), next_row);
    };
    look((int64_t)first * 32);
    for (int64_t k0 = (int64_t)first * 32; k0 < count; k0 += (int64_t)step * 32) {
        const int page = next_page, in_page = next_row;
        look(k0 + (int64_t)step * 32);
        float s = -INFINITY, vscale = 1.f;
        int64_t voff = 0;
        if (page >= 0) {
            const TC* row = keys + page * p.c.key_stride[0] + in_page * p.c.key_stride[2];
            voff = page * p.c.value_stride[0] + in_page * p.c.value_stride[2];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
            for (int d = 0; d < D; d += 8) {
                float v[8];
                load8<WIDE>(row + d, D - d, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i & 3] = fmaf(q(d + i), v[i], sum[i & 3]);
            }
            s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (sizeof(TC) == 1) {
                s *= p.c.key_scale[row_offset(p.c.key_scale_stride, page, head, in_page)];
                vscale = p.c.value_scale[row_offset(p.c.value_scale_stride, page, head, in_page)];
            }
        }
        const unsigned seen = __ballot_sync(kFull, page >= 0);
        if (seen == 0) continue;
        const float m = fmaxf(r.m, warp_max(s));
        const float base = m == -INFINITY ? 0.f : m;        // nothing but scores of -infinity so far
        const float alpha = exp2f(r.m - base);
        const float w = page >= 0 ? exp2f(s - base) : 0.f;
        r.m = m;
        r.l = r.l * alpha + warp_sum(w);
#pragma unroll
        for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c) r.acc[c] *= alpha;
        const float weight = page >= 0 && w != 0.f ? w * vscale : 0.f;
        const unsigned adds = __ballot_sync(kFull, page >= 0 && w != 0.f);
        constexpr int kRows = 4;                            // value rows in flight
#pragma unroll 2
        for (int i0 = 0; i0 < 32; i0 += kRows) {
            float v[kRows][FK_MAX_HEAD_DIM / 32];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int64_t off = __shfl_sync(kFull, voff, i0 + i);
#pragma unroll
                for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
                    v[i][c] = ((adds >> (i0 + i)) & 1u) && c * 32 + lane < D ? load_elem(values + off + c * 32 + lane) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const float wi = __shfl_sync(kFull, weight, i0 + i);
#pragma unroll
                for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c) r.acc[c] = fmaf(wi, v[i][c], r.acc[c]);
            }
        }
    }
}

// A kernel's shared-memory limit, set once per device (a call of the runtime each time costs a twentieth of a decode call's host time).
// `done` belongs to the kernel.
template <typename K>
inline cudaError_t allow_smem(K* kern, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Kernel for few query rows per key/value head (attention_few.cu).  need != null: only the workspace's size.
bool attention_few_supported(const AttnParams& p, int dtype, int max_query);
int attention_few(const AttnParams& p, int dtype, int max_query, size_t* need, cudaStream_t stream);
// Kernel for tiles of 256 query rows (attention_tile.cu).
bool attention_tile_supported(const AttnParams& p, int dtype);
int attention_tile(const AttnParams& p, int dtype, size_t* need, cudaStream_t stream);

}  // namespace fk
