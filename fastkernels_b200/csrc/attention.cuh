// Paged attention: what its kernels share.
#pragma once

#include <atomic>
#include <type_traits>

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

// Eight elements of a key or value row as they lie in memory: 16 bytes, 8 of codes.
template <typename TC>
struct Raw8 {
    static_assert(sizeof(TC) <= 2, "rows of 16-bit elements or codes");
    typename std::conditional<sizeof(TC) == 2, uint4, uint2>::type w;
    __device__ __forceinline__ void load(const TC* p, bool there) {
        w = {};
        if (there) w = *reinterpret_cast<const decltype(w)*>(p);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const { load8<true>(reinterpret_cast<const TC*>(&w), 8, v); }
};

// The sums of one row over its keys, held by a warp: lane l has the elements 8 l .. 8 l + 7 of acc.
struct RowSums {
    float m, l;
    float acc[8];
};

// A row that is computed again (row_again): one warp, one query row (lane l has the elements 8 l .. 8 l + 7 times scale * log2 e, zeros behind
// head_dim), 32 of the visible keys at a time.  One lane computes one key's score (no reduction per key; the query's elements go round by
// shuffles), then the value rows are added one at a time, eight columns per lane; four loads are in flight, which is what 64 registers
// hold.  Keys that are masked never enter any sum, whatever their rows hold.
template <typename TC>
__device__ __forceinline__ void warp_row(const AttnParams& p, const float (&q)[8], int seq, int head, int pos, RowSums& r) {
    const int lane = threadIdx.x & 31, D = p.c.head_dim;
    const int end = min(pos + 1, p.c.max_pages * p.c.page_size);       // positions that the table does not hold are not visible
    const int lo = window_start(p, pos), n_sinks = max(0, min(p.sinks, min(lo, end)));
    const int count = n_sinks + max(0, end - lo);
    r.m = -INFINITY;
    r.l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.acc[e] = 0.f;
    const TC* keys = reinterpret_cast<const TC*>(p.c.key) + head * p.c.key_stride[1];
    const TC* values = reinterpret_cast<const TC*>(p.c.value) + head * p.c.value_stride[1];
    for (int64_t k0 = 0; k0 < count; k0 += 32) {
        int page = -1, in_page = 0;
        if (k0 + lane < count) page = page_of(p.c, seq, (int)(k0 + lane < n_sinks ? k0 + lane : lo + k0 + lane - n_sinks), in_page);
        if (!__any_sync(kFull, page >= 0)) continue;
        const TC* row = keys + (page < 0 ? 0 : page * p.c.key_stride[0] + in_page * p.c.key_stride[2]);
        const int64_t voff = page < 0 ? 0 : page * p.c.value_stride[0] + in_page * p.c.value_stride[2];
        float s = 0.f;
        for (int d0 = 0; d0 < D; d0 += 32) {
            Raw8<TC> raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i].load(row + d0 + 8 * i, page >= 0 && d0 + 8 * i < D);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
                raw[i].values(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e & 3] = fmaf(__shfl_sync(kFull, q[e], d0 / 8 + i), v[e], sum[e & 3]);
            }
            s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        float vscale = 1.f;
        if (sizeof(TC) == 1 && page >= 0) {
            s *= p.c.key_scale[row_offset(p.c.key_scale_stride, page, head, in_page)];
            vscale = p.c.value_scale[row_offset(p.c.value_scale_stride, page, head, in_page)];
        }
        if (page < 0) s = -INFINITY;
        const float m = fmaxf(r.m, warp_max(s));
        const float base = m == -INFINITY ? 0.f : m;        // nothing but scores of -infinity so far
        const float alpha = exp2f(r.m - base);
        const float w = page >= 0 ? exp2f(s - base) : 0.f;
        r.m = m;
        r.l = r.l * alpha + warp_sum(w);
#pragma unroll
        for (int e = 0; e < 8; ++e) r.acc[e] *= alpha;
        const float weight = page >= 0 && w != 0.f ? w * vscale : 0.f;
        const unsigned adds = __ballot_sync(kFull, page >= 0 && w != 0.f);
        for (int i0 = 0; i0 < 32; i0 += 4) {
            Raw8<TC> raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i].load(values + __shfl_sync(kFull, voff, i0 + i) + 8 * lane, ((adds >> (i0 + i)) & 1u) && 8 * lane < D);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float one = __shfl_sync(kFull, weight, i0 + i);
                float v[8];
                raw[i].values(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) r.acc[e] = fmaf(one, v[e], r.acc[e]);
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
