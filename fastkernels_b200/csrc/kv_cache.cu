// Paged key/value cache: new tokens written (as they are, or as e4m3 codes with a scale per row) and read back.
//
// A row is one token's head_dim elements of one head.  Sixteen elements per lane (32 bytes of a 16-bit type: one access), ceil(head_dim
// / 16) lanes per row rounded up to a power of two; the row's maximum is one group-wide shuffle reduction.  Both kernels are streams of
// bytes, bound by HBM if enough of them are on their way: a block takes a few tokens with all heads, keys and values, looks their
// places up once (a search over the sequences and a read of the page table are four to eight dependent loads), and every thread then
// has kAhead pieces of rows in flight, unconverted.
//
// Codes: x * 448 / max must not be moved across the middle between two codes by a rounding, and for 16-bit rows many quotients lie
// exactly there.  q = x r with r = 1 / max, then q + (x - q max) r (one step of Newton's iteration with the exact residual of a
// fused multiply-add; P. Markstein, IBM J. Res. Dev. 34, 1990): where x / max is a number of few bits the step lands on it, since
// what it adds is off by 2^-24 of the residual only.  A divide per element costs three times as many instructions and bounds the
// kernel instead of HBM.  Elements of 24 bits leave quotients that round to such a middle without lying on it (a few in ten million): theirs
// are rounded to odd, the residual telling the side, so that the second rounding, to the code, sees where they were.

#include "kernels.cuh"
#include "kv_cache.cuh"

namespace fk {

int dtype_bytes(int dtype) { return dtype == FK_F32 ? 4 : dtype == FK_E4M3 ? 1 : 2; }

int check_cache(const fk_kv_cache& c) {
    if (c.pages < 1 || c.kv_heads < 1 || c.page_size < 1 || c.head_dim < 1 || c.head_dim > FK_MAX_HEAD_DIM) return FK_ERR_ARG;
    if (c.seqs < 0 || c.max_pages < 0 || c.table_stride < 0) return FK_ERR_ARG;
    if ((int64_t)c.max_pages * c.page_size > INT32_MAX - 1024) return FK_ERR_ARG;       // positions past a tile's end are still ints
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

constexpr int kRowThreads = 256;
constexpr int kAhead = 4;          // pieces of rows in flight per thread
constexpr int kMostTokens = 32;    // of a block
constexpr int kPiece = 16;         // elements of a lane

// A lane's sixteen elements as they lie in memory.
template <typename T>
struct Piece {
    uint4 w[sizeof(T)];
    __device__ __forceinline__ void values(float (&v)[kPiece]) const {
        float h[8];
        const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            load8<true>(e + 8 * i, 8, h);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[8 * i + k] = h[k];
        }
    }
    __device__ __forceinline__ void set(const float (&v)[kPiece]) {
        T* e = reinterpret_cast<T*>(w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float h[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
            store8<true>(e + 8 * i, 8, h);
        }
    }
};

// How a piece may be accessed.  whole: all 16 elements, 32 bytes at a time (16 of codes); halves: eight elements at a time; single: one by one.
enum Access { whole, halves, single };

__device__ __forceinline__ void ld32(const void* p, uint4& a, uint4& b) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ void st32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}

template <Access A, typename T>
__device__ __forceinline__ void load_piece(const T* p, int n, Piece<T>& r) {
    if (A == whole) {
        if (sizeof(T) == 1) r.w[0] = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i + 1 < (int)sizeof(T); i += 2) ld32(reinterpret_cast<const uint4*>(p) + i, r.w[i], r.w[i + 1]);
        return;
    }
    T* e = reinterpret_cast<T*>(r.w);
    if (A == halves) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (n > 8 * i) {
                if (sizeof(T) == 1) reinterpret_cast<uint2*>(r.w)[i] = reinterpret_cast<const uint2*>(p)[i];
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k) r.w[i * (sizeof(T) / 2) + k] = reinterpret_cast<const uint4*>(p)[i * (sizeof(T) / 2) + k];
            }
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
            if (i < n) e[i] = p[i];
    }
}
template <Access A, typename T>
__device__ __forceinline__ void store_piece(T* p, int n, const Piece<T>& r) {
    if (A == whole) {
        if (sizeof(T) == 1) *reinterpret_cast<uint4*>(p) = r.w[0];
#pragma unroll
        for (int i = 0; i + 1 < (int)sizeof(T); i += 2) st32(reinterpret_cast<uint4*>(p) + i, r.w[i], r.w[i + 1]);
        return;
    }
    const T* e = reinterpret_cast<const T*>(r.w);
    if (A == halves) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (n > 8 * i) {
                if (sizeof(T) == 1) reinterpret_cast<uint2*>(p)[i] = reinterpret_cast<const uint2*>(r.w)[i];
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(p)[i * (sizeof(T) / 2) + k] = r.w[i * (sizeof(T) / 2) + k];
            }
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
            if (i < n) p[i] = e[i];
    }
}

struct KvParams {
    fk_kv_cache c;
    fk_kv_rows r;
    int group_log2;                // lanes per row, as a power of two
    int block_tokens;
    uint32_t per_token_inverse;    // 2^32 / (2 kv_heads) + 1: quotients of row numbers below 2^16
};

struct RowAt {
    int token, head;
    bool value;
};

// Place of each of the block's tokens: page (-1: none; -2: behind the last sequence) and row in it.
__device__ __forceinline__ void look_up_tokens(const KvParams& p, int first, int tokens, int2* place) {
    for (int i = threadIdx.x; i < tokens; i += kRowThreads) {
        const RowPlace at = place_of_row(p.r.starts, p.c.lengths, p.c.seqs, p.r.rows, first + i);
        int in_page = 0;
        place[i].x = at.seq < 0 ? -2 : page_of(p.c, at.seq, at.pos, in_page);
        place[i].y = in_page;
    }
}

__device__ __forceinline__ RowAt row_at(const KvParams& p, int row) {
    const int per_token = 2 * p.c.kv_heads;
    RowAt a;
    a.token = (int)__umulhi((uint32_t)row, p.per_token_inverse);
    const int rest = row - a.token * per_token;
    a.value = rest >= p.c.kv_heads;
    a.head = a.value ? rest - p.c.kv_heads : rest;
    return a;
}

// x * 448 / most to 24 bits, rounded to odd where they do not hold it: the rounding to a code that follows sees on which side of a middle
// the quotient lies.
__device__ __forceinline__ void nearest_quotients(float most, float (&v)[kPiece]) {
    const float lift = most < 0x1p-40f ? 0x1p60f : 1.f;            // residuals stay above the least fp32 number
    const float b = most * lift * 0x1p-9f, inv = 1.0f / b;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
        const float y = v[i] * lift, x = y * 0.875f, rest = fmaf(y, 0.875f, -x), q0 = x * inv;
        const float q = fmaf(fmaf(-q0, b, x) + rest, inv, q0), r = fmaf(-q, b, x) + rest;
        const uint32_t bits = __float_as_uint(q);
        v[i] = r == 0.f || q == 0.f ? q : __uint_as_float(((r < 0.f) != (q < 0.f) ? bits - 1 : bits) | 1u);
    }
}

template <typename T, typename TC, Access A>
__global__ void __launch_bounds__(kRowThreads) kv_append_kernel(const __grid_constant__ KvParams p) {
    __shared__ int2 place[kMostTokens];
    pdl_trigger();
    pdl_wait();
    const int first = blockIdx.x * p.block_tokens, tokens = min(p.block_tokens, p.r.rows - first);
    const int rows = tokens * 2 * p.c.kv_heads, step = kRowThreads >> p.group_log2;
    const int d0 = (threadIdx.x & ((1 << p.group_log2) - 1)) * kPiece, n = min(kPiece, p.c.head_dim - d0);
    look_up_tokens(p, first, tokens, place);
    bool looked = false;
    for (int r0 = threadIdx.x >> p.group_log2; r0 - (int)(threadIdx.x >> p.group_log2) < rows; r0 += step * kAhead) {
        Piece<T> raw[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int row = r0 + a * step;
            raw[a] = Piece<T>{};
            if (row < rows && n > 0) {
                const RowAt at = row_at(p, row);
                const int64_t* from = at.value ? p.r.value_stride : p.r.key_stride;
                load_piece<A>(reinterpret_cast<const T*>(at.value ? p.r.value : p.r.key) + (first + at.token) * from[0] + at.head * from[1] + d0, n, raw[a]);
            }
        }
        if (!looked) __syncthreads();            // the first rows are on their way while the places are looked up
        looked = true;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int row = r0 + a * step;
            const RowAt at = row_at(p, row);
            const int2 to_page = row < rows ? place[at.token] : make_int2(-1, 0);
            const int64_t* to = at.value ? p.c.value_stride : p.c.key_stride;
            TC* cache = reinterpret_cast<TC*>(at.value ? p.c.value : p.c.key) + to_page.x * to[0] + at.head * to[1] + to_page.y * to[2] + d0;
            if constexpr (sizeof(TC) == 1) {
                float v[kPiece], most = 0.f;
                raw[a].values(v);
#pragma unroll
                for (int i = 0; i < kPiece; ++i) most = max_nan(most, fabsf(v[i]));
                for (int o = 1 << p.group_log2 >> 1; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(kFull, most, o));
                most = max_nan(most, 0x1p-100f);
                // 448 = 0.875 * 2^9: the factors are split so that nothing overflows
                const float b = most * 0x1p-9f, inv = 1.0f / b;
                uint32_t middle = 0xffffffffu;           // fp32 rows: steps from two below a middle between codes to the quotient next to it
                uint32_t least = 0xffffffffu;            // twice the bits of the least magnitude but zero, less 1
#pragma unroll
                for (int i = 0; i < kPiece; ++i) {
                    const float x = v[i] * 0.875f, q = x * inv;
                    v[i] = fmaf(fmaf(-q, b, x), inv, q);
                    if constexpr (sizeof(T) == 4) {
                        middle = min(middle, (__float_as_uint(v[i]) - 0x7fffeu) & 0xfffffu);
                        least = min(least, (__float_as_uint(v[i]) << 1) - 1u);
                    }
                }
                // off by two steps of 2^-23 at most.  Below 2^-6 the middles lie closer together
                if constexpr (sizeof(T) == 4)
                    if (middle < 5 || least < 0x78ffffffu || most < 0x1p-40f) {
                        raw[a].values(v);
                        nearest_quotients(most, v);
                    }
                if (to_page.x < 0) continue;
                if (d0 == 0) {
                    const int64_t* ts = at.value ? p.c.value_scale_stride : p.c.key_scale_stride;
                    (at.value ? p.c.value_scale : p.c.key_scale)[to_page.x * ts[0] + at.head * ts[1] + to_page.y * ts[2]] = most / 448.0f;
                }
                Piece<TC> codes;
                codes.set(v);
                if (n > 0) store_piece<A>(cache, n, codes);
            } else {
                if (to_page.x >= 0 && n > 0) store_piece<A>(cache, n, raw[a]);
            }
        }
    }
}

template <typename T, typename TC, Access A>
__global__ void __launch_bounds__(kRowThreads) kv_gather_kernel(const __grid_constant__ KvParams p) {
    __shared__ int2 place[kMostTokens];
    pdl_trigger();
    pdl_wait();
    const int first = blockIdx.x * p.block_tokens, tokens = min(p.block_tokens, p.r.rows - first);
    const int rows = tokens * 2 * p.c.kv_heads, step = kRowThreads >> p.group_log2;
    const int d0 = (threadIdx.x & ((1 << p.group_log2) - 1)) * kPiece, n = min(kPiece, p.c.head_dim - d0);
    look_up_tokens(p, first, tokens, place);
    __syncthreads();
    if (n <= 0) return;
    for (int r0 = threadIdx.x >> p.group_log2; r0 < rows; r0 += step * kAhead) {
        Piece<TC> raw[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int row = r0 + a * step;
            raw[a] = Piece<TC>{};
            scale[a] = 1.f;
            if (row >= rows) continue;
            const RowAt at = row_at(p, row);
            const int2 from_page = place[at.token];
            if (from_page.x < 0) continue;
            const int64_t* from = at.value ? p.c.value_stride : p.c.key_stride;
            load_piece<A>(reinterpret_cast<const TC*>(at.value ? p.c.value : p.c.key) + from_page.x * from[0] + at.head * from[1] + from_page.y * from[2] + d0, n, raw[a]);
            if (sizeof(TC) == 1) {
                const int64_t* sf = at.value ? p.c.value_scale_stride : p.c.key_scale_stride;
                scale[a] = (at.value ? p.c.value_scale : p.c.key_scale)[from_page.x * sf[0] + at.head * sf[1] + from_page.y * sf[2]];
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int row = r0 + a * step;
            const RowAt at = row_at(p, row);
            if (row >= rows || (place[at.token].x == -2 && !p.r.zero_rest)) continue;
            const int64_t* to = at.value ? p.r.value_stride : p.r.key_stride;
            T* out = reinterpret_cast<T*>(at.value ? p.r.value : p.r.key) + (first + at.token) * to[0] + at.head * to[1] + d0;
            if constexpr (sizeof(TC) == 1) {
                float v[kPiece];
                raw[a].values(v);
#pragma unroll
                for (int i = 0; i < kPiece; ++i) v[i] *= scale[a];
                Piece<T> wide;
                wide.set(v);
                store_piece<A>(out, n, wide);
            } else {
                store_piece<A>(out, n, raw[a]);
            }
        }
    }
}

static int check_rows(const fk_kv_cache& c, const fk_kv_rows& r) {
    if (r.rows < 0) return FK_ERR_ARG;
    if (r.dtype != FK_F32 && r.dtype != FK_BF16 && r.dtype != FK_F16) return FK_ERR_UNSUPPORTED;
    if (c.dtype != FK_E4M3 && c.dtype != r.dtype) return FK_ERR_UNSUPPORTED;
    if (r.rows > 0 && (!r.key || !r.value)) return FK_ERR_ARG;
    return FK_OK;
}

template <bool APPEND, typename T, typename TC, Access A>
static int launch_rows_by(const KvParams& p, cudaStream_t stream) {
    const int64_t blocks = ((int64_t)p.r.rows + p.block_tokens - 1) / p.block_tokens;
    auto kern = APPEND ? kv_append_kernel<T, TC, A> : kv_gather_kernel<T, TC, A>;
    FK_CUDA_OK(launch_pdl(kern, dim3((unsigned)blocks), dim3(kRowThreads), 0, stream, p), APPEND ? "kv append launch" : "kv gather launch");
    FK_LAUNCH_OK(APPEND ? "kv append launch" : "kv gather launch");
    return FK_OK;
}

template <bool APPEND, typename T, typename TC>
static int launch_rows(const KvParams& p, cudaStream_t stream) {
    // whether groups of `elements` elements lie on their own boundaries (32 bytes at most) in the rows and in the cache
    auto aligned = [&](int elements) {
        const int ra = elements * (int)sizeof(T) < 32 ? elements * (int)sizeof(T) : 32, ca = elements * (int)sizeof(TC) < 32 ? elements * (int)sizeof(TC) : 32;
        return p.c.head_dim % elements == 0 && groups_aligned(p.r.key, p.r.key_stride, 2, sizeof(T), ra) && groups_aligned(p.r.value, p.r.value_stride, 2, sizeof(T), ra) &&
               groups_aligned(p.c.key, p.c.key_stride, 3, sizeof(TC), ca) && groups_aligned(p.c.value, p.c.value_stride, 3, sizeof(TC), ca);
    };
    if (aligned(16)) return launch_rows_by<APPEND, T, TC, whole>(p, stream);
    if (aligned(8)) return launch_rows_by<APPEND, T, TC, halves>(p, stream);
    return launch_rows_by<APPEND, T, TC, single>(p, stream);
}

template <bool APPEND>
static int kv_rows(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) {
    if (cache == nullptr || rows == nullptr) return FK_ERR_ARG;
    int st = check_cache(*cache);
    if (st != FK_OK) return st;
    st = check_rows(*cache, *rows);
    if (st != FK_OK) return st;
    if (cache->kv_heads > FK_MAX_KV_HEADS) return FK_ERR_UNSUPPORTED;      // row numbers of a block stay below 2^16
    if (rows->rows == 0 || (cache->seqs == 0 && (APPEND || !rows->zero_rest))) return FK_OK;
    KvParams p{*cache, *rows, 0, 1, (uint32_t)((1ull << 32) / (2 * cache->kv_heads) + 1)};
    while ((kPiece << p.group_log2) < cache->head_dim) ++p.group_log2;
    // Tokens per block: as many as leave four blocks for every SM and a turn of the loop for a block
    const int64_t token_items = (int64_t)(2 * cache->kv_heads) << p.group_log2;
    while (p.block_tokens < kMostTokens && p.block_tokens * token_items < kRowThreads * kAhead && rows->rows / (2 * p.block_tokens) >= 4 * sm_count()) p.block_tokens *= 2;
    cudaStream_t s = (cudaStream_t)stream;
    if (cache->dtype == FK_E4M3) {
        if (rows->dtype == FK_BF16) return launch_rows<APPEND, __nv_bfloat16, __nv_fp8_e4m3>(p, s);
        if (rows->dtype == FK_F16) return launch_rows<APPEND, __half, __nv_fp8_e4m3>(p, s);
        return launch_rows<APPEND, float, __nv_fp8_e4m3>(p, s);
    }
    if (rows->dtype == FK_BF16) return launch_rows<APPEND, __nv_bfloat16, __nv_bfloat16>(p, s);
    if (rows->dtype == FK_F16) return launch_rows<APPEND, __half, __half>(p, s);
    return launch_rows<APPEND, float, float>(p, s);
}

}  // namespace fk

extern "C" {

int fk_kv_append(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) { return fk::kv_rows<true>(cache, rows, stream); }
int fk_kv_gather(const fk_kv_cache* cache, const fk_kv_rows* rows, void* stream) { return fk::kv_rows<false>(cache, rows, stream); }

}
