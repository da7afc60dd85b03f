// Where a token of a paged key/value cache lies, and loads and stores of eight elements of any supported type.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace fk {

// Rows of a call -> sequences.  starts may be null (row s belongs to sequence s).
struct RowPlace {
    int seq;       // -1: behind the last sequence
    int pos;       // position in the sequence; may lie outside of it if starts and lengths do not fit together
};

__device__ __forceinline__ RowPlace place_of_row(const int* __restrict__ starts, const int* __restrict__ lengths, int seqs, int rows, int row) {
    RowPlace r{-1, 0};
    if (starts == nullptr) {
        if (row >= seqs) return r;
        r.seq = row;
        r.pos = max(lengths[row], 0) - 1;
        return r;
    }
    // the first s with starts[s + 1] > row
    int lo = 0, hi = seqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    if (lo >= seqs || starts[lo] > row) return r;
    r.seq = lo;
    r.pos = max(lengths[lo], 0) - min(starts[lo + 1], rows) + row;        // at most lengths - 1, whatever the starts hold
    return r;
}

// Page of a position, or -1 if the table does not hold it or the entry is no page.
__device__ __forceinline__ int page_of(const fk_kv_cache& c, int seq, int pos, int& row_in_page) {
    if (pos < 0) return -1;
    const int column = pos / c.page_size;
    if (column >= c.max_pages) return -1;
    row_in_page = pos - column * c.page_size;
    const int page = c.page_table[(int64_t)seq * c.table_stride + column];
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

__device__ __forceinline__ int64_t row_offset(const int64_t (&stride)[3], int page, int head, int row) {
    return page * stride[0] + head * stride[1] + row * stride[2];
}

// Eight consecutive elements as fp32.  WIDE: the address is a multiple of the eight elements' size (at most 16 bytes);
// otherwise element by element, only the first n.
template <bool WIDE>
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
    if (WIDE) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}
template <bool WIDE>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int n, float (&v)[8]) {
    if (WIDE) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16lo(a.x); v[1] = bf16hi(a.x); v[2] = bf16lo(a.y); v[3] = bf16hi(a.y);
        v[4] = bf16lo(a.z); v[5] = bf16hi(a.z); v[6] = bf16lo(a.w); v[7] = bf16hi(a.w);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
    }
}
template <bool WIDE>
__device__ __forceinline__ void load8(const __half* p, int n, float (&v)[8]) {
    if (WIDE) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? __half2float(p[i]) : 0.f;
    }
}
// Four codes -> two pairs of fp16 (exact): one conversion per pair and nothing else; the conversion of the fp8 header's type costs four
// instructions per pair, which bound the kernels that read codes.
__device__ __forceinline__ void codes4_to_half(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
template <bool WIDE>
__device__ __forceinline__ void load8(const __nv_fp8_e4m3* p, int n, float (&v)[8]) {
    if (WIDE) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        uint32_t h[4];
        codes4_to_half(a.x, h[0], h[1]);
        codes4_to_half(a.y, h[2], h[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}

template <bool WIDE>
__device__ __forceinline__ void store8(float* p, int n, const float (&v)[8]) {
    if (WIDE) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = v[i];
    }
}
template <bool WIDE>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int n, const float (&v)[8]) {
    if (WIDE) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = __float2bfloat16_rn(v[i]);
    }
}
template <bool WIDE>
__device__ __forceinline__ void store8(__half* p, int n, const float (&v)[8]) {
    if (WIDE) {
        __half2 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = __float2half_rn(v[i]);
    }
}
template <bool WIDE>
__device__ __forceinline__ void store8(__nv_fp8_e4m3* p, int n, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    if (WIDE) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) reinterpret_cast<uint8_t*>(p)[i] = (uint8_t)(w[i >> 1] >> (8 * (i & 1)));
    }
}

int dtype_bytes(int dtype);
// Sizes, pointers, types and strides of a cache description; FK_OK or the status to return.
int check_cache(const fk_kv_cache& c);
// base and strides (in elements of `bytes` each) keep groups of eight elements on `align`-byte boundaries
bool groups_aligned(const void* base, const int64_t* stride, int n, int bytes, int align);

}  // namespace fk
