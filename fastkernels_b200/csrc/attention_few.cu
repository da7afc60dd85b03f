// Attention of few new tokens per sequence (decode) over a paged cache: a stream of the cache's bytes.
//
// The query rows that share a key/value head (heads of the group x tokens) are the 8 * NT columns of the products, the keys
// their rows: S^T[16 keys, columns] = K Q^T and O^T[dim, columns] += V^T P^T, both mma.sync m16n8k16 with fp32 sums.  At 8
// columns an instruction carries 512 bytes of the cache, so the tensor pipe is idle nine tenths of the time and what bounds the
// kernel is HBM; swapping the operands instead (queries as 16 rows) would double the instructions for nothing.  tcgen05 has no
// use here: its operands would have to be at least 64 rows.
//
// Every warp works alone: it takes 16 keys at a time through its own ring of shared-memory slots (cp.async, a slot of keys, then
// one of values), keeps its own running maximum and sum, and never waits for another warp.  The groups of 16 keys of all
// (sequence, head) items, in order, are dealt to the warps of the grid in equal contiguous runs, so uneven sequences need no
// schedule.  A run covers some items whole (written out at once) and at most two in part; the parts of a block's warps are joined at
// the block's end, what crosses blocks by attention_few_join_kernel, in key order, so the result does not depend on timing.
//
// 8-bit caches: the codes go to fp16 exactly; a query row is scaled by a power of two into fp16's range (exact for what is
// within 2^-14 of its largest element, to 2^-25 of it below), scores are multiplied by their key's scale, and the weights by
// their value's scale and a power of two per query row, which follows the largest such product that the row has met: no scale takes bits
// from the weights of rows that do not see it, or in which it has no weight.  Weights are rounded to the type of the products' operands, fp16 ones
// after a factor of 2^14 so that small ones keep their bits; sums stay in fp32.

#include <type_traits>

#include "attention_items.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace fk {

template <typename TC> struct FewOps {           // operand type of the products
    using T = TC;
    static constexpr bool kCodes = false;
};
template <> struct FewOps<__nv_fp8_e4m3> {
    using T = __half;
    static constexpr bool kCodes = true;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
// `bytes` (0 or all) are copied, the rest of the destination becomes zero
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int row, int group, int head, int page, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(group), "r"(head), "r"(page), "l"(policy)
        : "memory");
}

constexpr int kFewKeys = 16;                    // keys of one product, rows of a tensor copy
constexpr int kFewLeast = 2;                    // shortest run of a warp, in groups

template <int D, int NT, typename TC>
struct FewShape {
    static constexpr bool kCodes = FewOps<TC>::kCodes;
    static constexpr int kPitch = D * (int)sizeof(TC);                 // bytes of a row
    // Keys of a group: 32 where rows are short, so that what a group costs beside its bytes (waits, maxima, page numbers) is spread over more
    // of them (128 dimensions in 8 bits, 128 x 8000: 16 keys 335 us where 32 took 233; 241 to 256 on other machines)
    static constexpr int kTiles = kPitch <= 128 ? 2 : 1, kKeys = 16 * kTiles;
    static constexpr uint32_t kAllRows = 0xffffffffu >> (32 - kKeys);
    static constexpr int kSlot = kKeys * kPitch;
    static constexpr int kWarps = kCodes && NT == 1 && D <= 128 ? 12 : 8;      // as many as the registers hold
    static constexpr int kFit = 192 * 1024 / kWarps / kSlot;           // slots per warp in 192 KB
    static constexpr int kSlots = kFit > 8 ? 8 : kFit;
    static constexpr int kCols = 8 * NT;
    static constexpr int kPart = (D + 2) * kCols;                      // floats of a partial result: m, l per column, [column][D]
    // behind the ring, per slot: first key and row mask, scales of its rows, barrier
    static constexpr int kSide = 8 + (kCodes ? 4 * kKeys : 0) + 8;
    static constexpr int kRing = kWarps * kSlots * kSlot;
    static constexpr int kSmem = kRing + kWarps * kSlots * kSide + kWarps * 2 * (int)sizeof(PartHead) + kWarps * 16 + 16 + kWarps * 2 * 2 * kCols * 4 + kCols * 4;
    static_assert(kSlots >= 3, "a slot being read and two on their way");
    static_assert(kSmem <= 227 * 1024, "shared memory of a block");
};

// Byte of a slot at which 16-byte chunk `chunk` of row `row` is kept: the layout of a tensor copy with 128-byte swizzle.  ldmatrix
// reads eight rows of one chunk; with codes, a quarter of a warp reads chunks 0..3 (or 4..7) of two key rows that differ in bit 2, or
// two neighbouring chunks of four value rows that differ in bits 1 and 2 (key_row below): no conflicts.  Rows of 64 bytes: two reads
// of the values for one.
template <int D, typename TC>
__device__ __forceinline__ int slot_at(int row, int chunk) {
    if (D * sizeof(TC) >= 128) return (chunk >> 3) * (16 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
    return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// Key (row of the group) of row i < 8 of S^T, + 8 for the others.
template <typename TC>
__device__ __forceinline__ int key_row(int i) { return FewOps<TC>::kCodes ? ((i & 6) ^ ((i & 1) << 2)) | (i & 1) : i; }

// Column n of an item joined from `count` parts, by one warp: lane l has dimensions 4 l .. 4 l + 3 (and 128 more each), or 2 l, 2 l + 1
// at 64.  part(i) is the address of the i-th part.
template <int D>
struct Joined {
    static constexpr int kVec = D >= 128 ? 4 : 2, kParts = D / (32 * kVec);
    float m, l, acc[kParts][kVec];
    __device__ __forceinline__ static int dim(int lane, int c, int e) { return c * 32 * kVec + lane * kVec + e; }
    template <int COLS, typename Part>
    __device__ __forceinline__ void join(const Part& part, int first, int count, int step, int n) {
        const int lane = threadIdx.x & 31;
        m = -INFINITY;
        for (int i = first + lane * step; i < count; i += 32 * step) m = fmaxf(m, part(i)[n]);
        m = warp_max(m);
        const float base = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int e = 0; e < kVec; ++e) acc[c][e] = 0.f;
#pragma unroll 4
        for (int i = first; i < count; i += step) {
            const float* one = part(i);
            const float weight = exp2_fast(one[n] - base);
            l = fmaf(weight, one[COLS + n], l);
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
                const float* from = one + 2 * COLS + n * D + dim(lane, c, 0);
                float v[kVec];
                if (kVec == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(from);
                    v[0] = f.x; v[1] = f.y; v[kVec - 2] = f.z; v[kVec - 1] = f.w;
                } else {
                    const float2 f = *reinterpret_cast<const float2*>(from);
                    v[0] = f.x; v[1] = f.y;
                }
#pragma unroll
                for (int e = 0; e < kVec; ++e) acc[c][e] = fmaf(weight, v[e], acc[c][e]);
            }
        }
    }
    // the finished row
    template <typename T, typename TC>
    __device__ __forceinline__ void finish(const AttnParams& p, const PartHead& h, int n) const {
        const int lane = threadIdx.x & 31, tok = n / p.group, row = h.first_row + tok, qh = h.head * p.group + n - tok * p.group;
        T* out = reinterpret_cast<T*>(p.out) + (int64_t)row * p.os[0] + (int64_t)qh * p.os[1];
        bool odd = false;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float v = l == 0.f ? 0.f : acc[c][e] / l;
                odd |= l == l && !(fabsf(v) < INFINITY);
                store_elem(out + dim(lane, c, e), v);
            }
        if (h.tokens > 1 && __any_sync(kFull, odd)) {
            __syncwarp();
            row_again<T, TC>(p, h.seq, h.first_row, h.pos0, h.tokens, tok, qh);
        }
    }
};

// TMA: the 16 rows of a group lie in one page and come by one tensor copy (and one bulk copy of their scales); else by cp.async.
template <int D, int NT, typename T, typename TC, bool TMA>
__global__ void __launch_bounds__(32 * FewShape<D, NT, TC>::kWarps, 1) attention_few_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap key_map,
                                                                                         const __grid_constant__ CUtensorMap value_map) {
    using S = FewShape<D, NT, TC>;
    using OT = typename FewOps<TC>::T;
    constexpr bool kCodes = S::kCodes;
    constexpr int kMT = D / 16, kSlots = S::kSlots;
    constexpr float kShift = std::is_same<OT, __half>::value ? 14.f : 0.f;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kSlots * S::kSlot;
    unsigned char* side = smem + S::kRing;
    uint64_t* landed = reinterpret_cast<uint64_t*>(side) + warp * kSlots;                                               // tensor copies' barriers
    int2* meta = reinterpret_cast<int2*>(side + S::kWarps * kSlots * 8) + warp * kSlots;
    float* scales = reinterpret_cast<float*>(side + S::kWarps * kSlots * 16) + warp * kSlots * S::kKeys;                // codes
    PartHead* warp_heads = reinterpret_cast<PartHead*>(side + S::kWarps * kSlots * S::kSide);
    int64_t* scratch = reinterpret_cast<int64_t*>(warp_heads + S::kWarps * 2);
    int* abort_flag = reinterpret_cast<int*>(scratch + 2 * S::kWarps);
    int* odd_column = abort_flag + 4;
    float* stats = reinterpret_cast<float*>(odd_column + S::kCols);         // [2 warps' parts][m, l per column]
    int64_t* upto = reinterpret_cast<int64_t*>(smem);              // over the ring, before its first copy
    const int room = S::kRing / 8;
    if (TMA) {
        if (lane == 0) {
            for (int i = 0; i < kSlots; ++i) mbar_init(&landed[i], 1);
            mbar_init_fence();
        }
        __syncwarp();
    }
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        if (TMA) {
            prefetch_tensormap(&key_map);
            prefetch_tensormap(&value_map);
        }
    }
    pdl_trigger();
    pdl_wait();

    Runs runs{plan_tiles<S::kKeys>(p, scratch, upto, room), (int64_t)gridDim.x * S::kWarps, kFewLeast};
    const int64_t me = (int64_t)blockIdx.x * S::kWarps + warp;
    // workspace: heads of the blocks' parts, blocks' parts, warps' parts
    PartHead* block_heads = reinterpret_cast<PartHead*>(p.part) + blockIdx.x * 2;
    float* block_parts = p.part + gridDim.x * 2 * (sizeof(PartHead) / 4) + (int64_t)blockIdx.x * 2 * S::kPart;
    float* warp_parts = p.part + gridDim.x * 2 * (sizeof(PartHead) / 4) + ((int64_t)gridDim.x + (int64_t)blockIdx.x * S::kWarps) * 2 * S::kPart;
    PartHead* heads = warp_heads + warp * 2;
    float* parts = warp_parts + warp * 2 * S::kPart;
    const int64_t run0 = runs.begin(me), run1 = runs.begin(me + 1);
    if (lane < 2) heads[lane].begins = heads[lane].ends = -1;
    if (threadIdx.x < 2) block_heads[threadIdx.x].begins = block_heads[threadIdx.x].ends = -1;
    __syncwarp();

    ItemCursor<S::kKeys> cur, ahead;
    if (run0 < run1) locate(p, run0, upto, room, cur);
    if (TMA) fence_async_proxy();                // every thread's accesses to the plan, before copies of the other proxy write there
    __syncthreads();                             // the plan's memory is the ring's from here on
    ahead = cur;

    const uint64_t policy = l2_evict_first_policy();     // a row of the cache is read once per call

    // ---- issue side: keys and values of one group after the other into the ring
    int64_t left = run1 - run0;
    int page = -1, in_page = 0;                  // of this lane's row of the next group; tensor copies: of the first of its 16 rows
    bool seen = false;                           // some row sees this lane's key
    int64_t koff = -1, voff = -1;                // bytes; cp.async only
    int issue_slot = 0;
    auto look = [&] {                            // the page table is read one group ahead of its use
        page = -1;
        seen = false;
        if (left <= 0) return;
        const int j = ahead.key0() + (lane & (S::kKeys - 1));
        seen = ahead.some_row_sees(p, j);
        if (TMA || seen) page = page_of(p.c, ahead.seq, TMA ? j & ~15 : j, in_page);
    };
    auto issue = [&](bool values) {
        if (left > 0) {
            const uint32_t base = ring + issue_slot * S::kSlot;
            if (!values) {
                if (!TMA) {
                    koff = page < 0 ? -1 : row_offset(p.c.key_stride, page, ahead.head, in_page) * (int64_t)sizeof(TC);
                    voff = page < 0 ? -1 : row_offset(p.c.value_stride, page, ahead.head, in_page) * (int64_t)sizeof(TC);
                }
                const unsigned rows = __ballot_sync(kFull, page >= 0 && seen) & S::kAllRows;
                if (lane == 0) meta[issue_slot] = make_int2(ahead.key0(), (int)rows);
            }
            if (TMA) {
                uint64_t* bar = &landed[issue_slot];
                const unsigned there = __ballot_sync(kFull, page >= 0);
                if (lane == 0) mbar_expect_tx(bar, S::kSlot + (kCodes ? 64 * ((there & 1) + (S::kTiles > 1 ? (there >> 16) & 1 : 0)) : 0));
                if ((lane & 15) == 0 && lane < S::kKeys) {
                    tma_load_5d(base + lane * 128, values ? &value_map : &key_map, 0, in_page, 0, ahead.head, page < 0 ? p.c.pages : page, bar, policy);
                    if (kCodes && page >= 0)
                        bulk_load(scales + issue_slot * S::kKeys + lane,
                                  (values ? p.c.value_scale : p.c.key_scale) + row_offset(values ? p.c.value_scale_stride : p.c.key_scale_stride, page, ahead.head, in_page), 64, bar);
                }
                __syncwarp();
            } else {
                const char* from = reinterpret_cast<const char*>(values ? p.c.value : p.c.key);
                constexpr int kChunks = S::kPitch / 16, kAtOnce = 32 / kChunks;
#pragma unroll
                for (int i = 0; i < S::kKeys / kAtOnce; ++i) {
                    const int row = i * kAtOnce + lane / kChunks, chunk = lane % kChunks;
                    const int64_t off = __shfl_sync(kFull, values ? voff : koff, row);
                    copy16(base + slot_at<D, TC>(row, chunk), off < 0 ? from : from + off + chunk * 16, off < 0 ? 0 : 16);
                }
                if (kCodes && lane < S::kKeys) {
                    const float* s = values ? p.c.value_scale : p.c.key_scale;
                    copy4(smem_u32(scales + issue_slot * S::kKeys + lane),
                          page < 0 ? s : s + (values ? row_offset(p.c.value_scale_stride, page, ahead.head, in_page) : row_offset(p.c.key_scale_stride, page, ahead.head, in_page)),
                          page < 0 ? 0 : 4);
                }
            }
            if (values) {
                --left;
                if (++ahead.k >= ahead.span.count && left > 0) ahead.next_item(p);
                look();
            }
        }
        if (!TMA) asm volatile("cp.async.commit_group;" ::: "memory");
        if (++issue_slot == kSlots) issue_slot = 0;
    };
    if (run0 < run1) look();
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) issue(i & 1);
    int slot = 0;
    uint32_t phase = 0;
    bool zeroed = false;                         // threads wrote to the slot that is read
    // the oldest slot has landed for the whole warp, and the one before it is free
    auto next_slot = [&](bool issue_values) {
        if (TMA) {
            if (left >= 0 && !warp_wait(&landed[slot], phase, abort_flag, p.wait_cycles)) {
                left = -1;                       // nothing more is issued or waited for
                *abort_flag = 1;
            }
        } else asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 2) : "memory");
        if (TMA && zeroed) fence_async_proxy();
        zeroed = false;
        __syncwarp();
        issue(issue_values);
        const int now = slot;
        if (++slot == kSlots) { slot = 0; phase ^= 1; }
        return now;
    };

    const int row_lo = key_row<TC>(g), row_hi = row_lo + 8;      // this thread's key rows of S^T
    int64_t at = run0;
    while (at < run1) {
        const int steps = (int)min((int64_t)(cur.span.count - cur.k), run1 - at);
        const bool begins = cur.k == 0, ends = cur.k + steps == cur.span.count;
        const int first_row = cur.first_row(p), tokens = cur.tokens(p), cols = tokens * p.group;
        // ---- query fragments
        uint32_t qf[NT][kMT][2];
        float qscale[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int n = nt * 8 + g;
            const int tok = n / p.group;
            const T* q = reinterpret_cast<const T*>(p.query) + (int64_t)(first_row + (n < cols ? tok : 0)) * p.qs[0] +
                         (int64_t)(cur.head * p.group + (n < cols ? n - tok * p.group : 0)) * p.qs[1];
#pragma unroll
            for (int kk = 0; kk < kMT; ++kk)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = kCodes ? ((kk >> 2) * 4 + t) * 16 + (kk & 3) * 4 + 2 * h : kk * 16 + 2 * t + 8 * h;
                    qf[nt][kk][h] = n < cols ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                }
            if (kCodes) {
                float most = 0.f;
#pragma unroll
                for (int kk = 0; kk < kMT; ++kk)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const T* two = reinterpret_cast<const T*>(&qf[nt][kk][h]);
                        most = fmaxf(most, fmaxf(fabsf(to_float(two[0])), fabsf(to_float(two[1]))));
                    }
                most = fmaxf(most, __shfl_xor_sync(kFull, most, 1));
                most = fmaxf(most, __shfl_xor_sync(kFull, most, 2));
                const int e = row_exponent(most);
                const float down = ldexpf(1.f, -e);
#pragma unroll
                for (int kk = 0; kk < kMT; ++kk)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const T* two = reinterpret_cast<const T*>(&qf[nt][kk][h]);
                        qf[nt][kk][h] = pack2(to_float(two[0]) * down, to_float(two[1]) * down, __half{});
                    }
                const float up = ldexpf(p.scale_log2, e);
                qscale[nt][0] = __shfl_sync(kFull, up, 8 * t);
                qscale[nt][1] = __shfl_sync(kFull, up, 8 * t + 4);
            } else {
                qscale[nt][0] = qscale[nt][1] = p.scale_log2;
            }
        }
        float acc[NT][kMT][4], m[NT][2], l[NT][2];
        // codes, per column: the largest weight x value scale met so far, and the power of two that such products are multiplied by before they
        // are rounded; it only moves where one exceeds 2^15 or the maximum of the scores has risen
        float most_out[NT][2], up_out[NT][2];
        auto power_for = [](float product) { return __int_as_float(min(max(253 - (__float_as_int(product) >> 23), 15), 239) << 23); };     // -> [1/2, 1)
        auto inverse = [](float power) { return __int_as_float(0x7f000000 - __float_as_int(power)); };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < kMT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
            most_out[nt][0] = most_out[nt][1] = 0.f;
            up_out[nt][0] = up_out[nt][1] = 0x1p112f;
        }
        const int sure_lo = window_start(p, cur.pos1);        // keys that every token of the item sees: sure_lo .. pos0

        for (int step = 0; step < steps; ++step) {
            // ---- scores
            const int ks = next_slot((kSlots - 1) & 1);
            const uint32_t kbase = ring + ks * S::kSlot;
            const int2 what = meta[ks];
            float s[S::kTiles][NT][4];
#pragma unroll
            for (int kt = 0; kt < S::kTiles; ++kt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[kt][nt][0] = s[kt][nt][1] = s[kt][nt][2] = s[kt][nt][3] = 0.f;
                if (kCodes) {
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        const uint4 lo = lds16(kbase + slot_at<D, TC>(row_lo + 16 * kt, 4 * i + t)), hi = lds16(kbase + slot_at<D, TC>(row_hi + 16 * kt, 4 * i + t));
                        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t a[4];
                            codes4_to_half(wl[j], a[0], a[2]);
                            codes4_to_half(wh[j], a[1], a[3]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma16816(s[kt][nt], a, qf[nt][4 * i + j], OT{});
                        }
                    }
                    const float k0 = scales[ks * S::kKeys + row_lo + 16 * kt], k1 = scales[ks * S::kKeys + row_hi + 16 * kt];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        s[kt][nt][0] *= qscale[nt][0] * k0; s[kt][nt][1] *= qscale[nt][1] * k0;
                        s[kt][nt][2] *= qscale[nt][0] * k1; s[kt][nt][3] *= qscale[nt][1] * k1;
                    }
                } else {
                    float s2[NT][4];                  // two chains of products
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s2[nt][0] = s2[nt][1] = s2[nt][2] = s2[nt][3] = 0.f;
                    const int row = (lane & 15) + 16 * kt;
#pragma unroll
                    for (int kk = 0; kk < kMT; ++kk) {
                        uint32_t a[4];
                        ldmatrix4(a, kbase + slot_at<D, TC>(row, 2 * kk + (lane >> 4)));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(kk & 1 ? s2[nt] : s[kt][nt], a, qf[nt][kk], OT{});
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kt][nt][i] = (s[kt][nt][i] + s2[nt][i]) * p.scale_log2;
                }
            }
            // ---- masks: rows that are not there, and keys that only some of the tokens see
            const bool all = tokens == 1 || (what.x + S::kKeys - 1 <= cur.pos0 && (p.window == 0 || what.x >= sure_lo || what.x + S::kKeys <= p.sinks));
            const bool all_rows = (uint32_t)what.y == S::kAllRows;
            if (!all_rows || !all) {
#pragma unroll
                for (int kt = 0; kt < S::kTiles; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = (i < 2 ? row_lo : row_hi) + 16 * kt, n = nt * 8 + 2 * t + (i & 1);
                            if (!(((uint32_t)what.y >> row) & 1) || (!all && !sees(p, cur.pos0 + n / p.group, what.x + row))) s[kt][nt][i] = -INFINITY;
                        }
            }
            // ---- running maximum, weights
            bool grew = false;
            float mn[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
                    if (S::kTiles > 1) x = fmaxf(x, fmaxf(s[S::kTiles - 1][nt][c], s[S::kTiles - 1][nt][c + 2]));
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 16));
                    mn[nt][c] = fmaxf(m[nt][c], x);
                    grew |= mn[nt][c] > m[nt][c];
                }
            if (__any_sync(kFull, grew)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float a = mn[nt][c] > m[nt][c] ? exp2_fast(m[nt][c] - mn[nt][c]) : 1.f;
                        m[nt][c] = mn[nt][c];
                        l[nt][c] *= a;
                        float factor = a;
                        if (kCodes) {
                            most_out[nt][c] *= a;
                            if (most_out[nt][c] > 0.f) {
                                const float power = power_for(most_out[nt][c]);
                                factor = a * (power * inverse(up_out[nt][c]));
                                up_out[nt][c] = power;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < kMT; ++i) { acc[nt][i][c] *= factor; acc[nt][i][c + 2] *= factor; }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float base = m[nt][c] == -INFINITY ? 0.f : m[nt][c] - kShift;
#pragma unroll
                    for (int kt = 0; kt < S::kTiles; ++kt) {
                        s[kt][nt][c] = exp2_fast(s[kt][nt][c] - base);
                        s[kt][nt][c + 2] = exp2_fast(s[kt][nt][c + 2] - base);
                        l[nt][c] += s[kt][nt][c] + s[kt][nt][c + 2];
                    }
                }
            // ---- values
            const int vs = next_slot(((kSlots - 1) & 1) ^ 1);
            const uint32_t vbase = ring + vs * S::kSlot;
            if (TMA && !all_rows) {
                // rows that nobody may see can hold anything, and 0 * infinity is no zero
                for (int i = lane; i < S::kSlot / 16; i += 32) {
                    const int row = (i >> 3) & (S::kKeys - 1);
                    if (!(((uint32_t)what.y >> row) & 1)) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vbase + i * 16), "r"(0) : "memory");
                }
                __syncwarp();
                zeroed = true;
            }
            if (kCodes) {
                float v[S::kTiles][2];
#pragma unroll
                for (int kt = 0; kt < S::kTiles; ++kt) {
                    v[kt][0] = scales[vs * S::kKeys + row_lo + 16 * kt];
                    v[kt][1] = scales[vs * S::kKeys + row_hi + 16 * kt];
                    if (!all_rows) {
                        if (!(((uint32_t)what.y >> (row_lo + 16 * kt)) & 1)) v[kt][0] = 0.f;
                        if (!(((uint32_t)what.y >> (row_hi + 16 * kt)) & 1)) v[kt][1] = 0.f;
                    }
                }
                bool over = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int kt = 0; kt < S::kTiles; ++kt)
                            over |= fmaxf(fabsf(s[kt][nt][c] * up_out[nt][c] * v[kt][0]), fabsf(s[kt][nt][c + 2] * up_out[nt][c] * v[kt][1])) > 0x1p15f;
                if (__any_sync(kFull, over)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = most_out[nt][c];
#pragma unroll
                            for (int kt = 0; kt < S::kTiles; ++kt)
                                x = fmaxf(x, fmaxf(fabsf(s[kt][nt][c] * 0x1p-14f * v[kt][0]), fabsf(s[kt][nt][c + 2] * 0x1p-14f * v[kt][1])));
                            x = fmaxf(x, __shfl_xor_sync(kFull, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(kFull, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(kFull, x, 16));
                            if (x == 0.f) continue;
                            most_out[nt][c] = x;
                            const float power = power_for(x), factor = power * inverse(up_out[nt][c]);
                            up_out[nt][c] = power;
#pragma unroll
                            for (int i = 0; i < kMT; ++i) { acc[nt][i][c] *= factor; acc[nt][i][c + 2] *= factor; }
                        }
                }
#pragma unroll
                for (int kt = 0; kt < S::kTiles; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kt][nt][i] = s[kt][nt][i] * up_out[nt][i & 1] * v[kt][i >> 1];
            }
#pragma unroll
            for (int kt = 0; kt < S::kTiles; ++kt) {
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    pf[nt][0] = transpose8x8(pack2(s[kt][nt][0], s[kt][nt][1], OT{}));
                    pf[nt][1] = transpose8x8(pack2(s[kt][nt][2], s[kt][nt][3], OT{}));
                }
                if (kCodes) {
                    constexpr int kUnits = D >= 128 ? D / 128 : 1, kWords = D >= 128 ? 4 : 2;
#pragma unroll
                    for (int u = 0; u < kUnits; ++u) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = key_row<TC>(2 * t + (i & 1)) + 4 * (i & 2) + 16 * kt;
                            if (D >= 128) {
                                const uint4 x = lds16(vbase + slot_at<D, TC>(row, g + 8 * u));
                                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                            } else {
                                const uint2 x = lds8(vbase + slot_at<D, TC>(row, g >> 1) + (g & 1) * 8);
                                w[i][0] = x.x; w[i][1] = x.y;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < kWords; ++j) {
                            uint32_t both[2][4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) codes4_to_half(w[i][j], both[0][i], both[1][i]);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t (&c)[4] = both[h];
                                const uint32_t a[4] = {__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[0], c[1], 0x7632), __byte_perm(c[2], c[3], 0x5410),
                                                       __byte_perm(c[2], c[3], 0x7632)};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][u * 8 + j * 2 + h], a, pf[nt], OT{});
                            }
                        }
                    }
                } else {
                    const int row = (lane & 7) + ((lane >> 4) << 3) + 16 * kt;
#pragma unroll
                    for (int i = 0; i < kMT; ++i) {
                        uint32_t a[4];
                        ldmatrix4_trans(a, vbase + slot_at<D, TC>(row, 2 * i + ((lane >> 3) & 1)));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][i], a, pf[nt], OT{});
                    }
                }
            }
        }

        // ---- the item's result, or this run's part of it.  acc[.][i][c + 2 h] is column 2t + c at dimension dim_of(i, h)
        auto dim_of = [&](int i, int h) { return kCodes ? (D >= 128 ? ((i >> 3) * 8 + g) * 16 + (i & 7) * 2 + h : g * 8 + i * 2 + h) : i * 16 + g + 8 * h; };
        auto unit = [&](int nt, int c) { return kCodes ? inverse(up_out[nt][c]) : 1.f; };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[nt][c] += __shfl_xor_sync(kFull, l[nt][c], 4);
                l[nt][c] += __shfl_xor_sync(kFull, l[nt][c], 8);
                l[nt][c] += __shfl_xor_sync(kFull, l[nt][c], 16);
                if (TMA && left < 0) l[nt][c] = NAN;       // a copy that never came: no number is right
            }
        if (begins && ends) {
            bool odd = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n = nt * 8 + 2 * t + c;
                    if (n >= cols) continue;
                    const int tok = n / p.group;
                    T* out = reinterpret_cast<T*>(p.out) + (int64_t)(first_row + tok) * p.os[0] + (int64_t)(cur.head * p.group + n - tok * p.group) * p.os[1];
                    const float inv = l[nt][c] == 0.f ? 0.f : unit(nt, c) / l[nt][c];
#pragma unroll
                    for (int i = 0; i < kMT; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float v = l[nt][c] == 0.f ? 0.f : acc[nt][i][c + 2 * h] * inv;
                            odd |= l[nt][c] == l[nt][c] && !(fabsf(v) < INFINITY);
                            store_elem(out + dim_of(i, h), v);
                        }
                }
            if (tokens > 1 && __any_sync(kFull, odd)) {
                __syncwarp();
                for (int n = 0; n < cols; ++n) row_again<T, TC>(p, cur.seq, first_row, cur.pos0, tokens, n / p.group, cur.head * p.group + n % p.group);
            }
        } else {
            // parts are kept without the weights' factor: beside it, sums of large values would end as infinities before the division
            constexpr float kUnshift = std::is_same<OT, __half>::value ? 0x1p-14f : 1.f;
            const int which = at == run0 ? 0 : 1;
            float* part = parts + which * S::kPart;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n = nt * 8 + 2 * t + c;
                    if (n >= cols) continue;
                    if (g == 0) {
                        float* st = stats + (warp * 2 + which) * 2 * S::kCols;
                        st[n] = m[nt][c];
                        st[S::kCols + n] = l[nt][c] * kUnshift;
                    }
#pragma unroll
                    for (int i = 0; i < kMT; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) part[2 * S::kCols + n * D + dim_of(i, h)] = acc[nt][i][c + 2 * h] * (unit(nt, c) * kUnshift);
                }
            if (lane == 0)
                heads[which] = PartHead{first_row, tokens, cur.head, cur.seq, cur.pos0, begins, ends, runs.worker_of(at - cur.k + cur.span.count - 1) / S::kWarps};
        }
        at += steps;
        if (at < run1) cur.next_item(p);
    }

    if (TMA && *reinterpret_cast<volatile int*>(abort_flag)) linger();       // copies still on their way to this block
    // ---- the parts of the block's warps: one that does not begin its item continues the one before it.  All threads take four
    // dimensions of a column each, so that a part costs one round of loads
    if (threadIdx.x < S::kCols) odd_column[threadIdx.x] = 0;
    __syncthreads();
    int group = -1;
    for (int e = 0; e < 2 * S::kWarps;) {
        if (warp_heads[e].begins < 0) { ++e; continue; }
        ++group;
        const int first = e;
        int last = e, count = 1;
        for (int f = e + 1; f < 2 * S::kWarps; ++f) {
            if (warp_heads[f].begins < 0) continue;
            if (warp_heads[f].begins == 1) break;
            last = f;
            ++count;
        }
        e = last + 1;
        const PartHead h = warp_heads[first];
        const bool begins = h.begins == 1, ends = warp_heads[last].ends == 1;
        // the first part may be either of its warp's two, all others are the first of theirs
        auto entry = [&](int i) { return i == 0 ? first : (first / 2 + i) * 2; };
        const int cols = h.tokens * p.group;
        float* to = block_parts + (group == 0 ? 0 : 1) * S::kPart;
        for (int i = threadIdx.x; i < cols * (D / 4); i += 32 * S::kWarps) {
            const int n = i / (D / 4), d = (i - n * (D / 4)) * 4;
            float m = -INFINITY, l = 0.f;
            for (int k = 0; k < count; ++k) m = fmaxf(m, stats[entry(k) * 2 * S::kCols + n]);
            const float base = m == -INFINITY ? 0.f : m;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int k = 0; k < count; ++k) {
                const float* st = stats + entry(k) * 2 * S::kCols + n;
                const float4 v = *reinterpret_cast<const float4*>(warp_parts + entry(k) * (int64_t)S::kPart + 2 * S::kCols + n * D + d);
                const float weight = exp2_fast(st[0] - base);
                l = fmaf(weight, st[S::kCols], l);
                acc.x = fmaf(weight, v.x, acc.x); acc.y = fmaf(weight, v.y, acc.y); acc.z = fmaf(weight, v.z, acc.z); acc.w = fmaf(weight, v.w, acc.w);
            }
            if (begins && ends) {
                const int tok = n / p.group;
                T* out = reinterpret_cast<T*>(p.out) + (int64_t)(h.first_row + tok) * p.os[0] + (int64_t)(h.head * p.group + n - tok * p.group) * p.os[1] + d;
                const float v[4] = {acc.x, acc.y, acc.z, acc.w};
                bool odd = false;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float r = l == 0.f ? 0.f : v[x] / l;
                    odd |= l == l && !(fabsf(r) < INFINITY);
                    store_elem(out + x, r);
                }
                if (odd && h.tokens > 1) odd_column[n] = 1;
            } else {
                if (d == 0) { to[n] = m; to[S::kCols + n] = l; }
                *reinterpret_cast<float4*>(to + 2 * S::kCols + n * D + d) = acc;
            }
        }
        if (begins && ends && h.tokens > 1) {
            __syncthreads();                     // the rows are written, then those that are not finite once more
            for (int n = warp; n < cols; n += S::kWarps) {
                const bool odd = odd_column[n] != 0;
                __syncwarp();
                if (odd) row_again<T, TC>(p, h.seq, h.first_row, h.pos0, h.tokens, n / p.group, h.head * p.group + n % p.group);
                if (lane == 0) odd_column[n] = 0;
            }
            __syncthreads();
        }
        if (!(begins && ends) && threadIdx.x == 0) {
            PartHead b = h;
            b.begins = begins;
            b.ends = ends;
            block_heads[group == 0 ? 0 : 1] = b;
        }
    }
}

// Joins the parts of one item from several blocks: a block per (block of the grid above whose run has the item's beginning, column).
constexpr int kJoinWarps = 4;

template <int D, int NT, typename T, typename TC>
__global__ void __launch_bounds__(32 * kJoinWarps) attention_few_join_kernel(const __grid_constant__ AttnParams p) {
    using S = FewShape<D, NT, TC>;
    __shared__ float sums[kJoinWarps][D + 2];
    pdl_trigger();
    pdl_wait();
    if (blockIdx.y == 0) zero_blind_rows<T>(p);
    const PartHead* heads = reinterpret_cast<const PartHead*>(p.part);
    const float* parts = p.part + gridDim.x * 2 * (sizeof(PartHead) / 4);
    const int w0 = blockIdx.x, n = blockIdx.y;
    int which = -1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (heads[2 * w0 + i].begins == 1 && heads[2 * w0 + i].ends == 0) which = i;
    if (which < 0) return;
    const PartHead h = heads[2 * w0 + which];
    if (n >= h.tokens * p.group) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = h.last - w0 + 1;
    auto part = [&](int i) { return parts + (int64_t)(i == 0 ? 2 * w0 + which : 2 * (w0 + i)) * S::kPart; };
    Joined<D> j;
    j.template join<S::kCols>(part, warp, count, kJoinWarps, n);
    if (count > 1) {                             // the warps' shares, in order
        if (lane == 0) { sums[warp][D] = j.m; sums[warp][D + 1] = j.l; }
#pragma unroll
        for (int c = 0; c < Joined<D>::kParts; ++c)
#pragma unroll
            for (int x = 0; x < Joined<D>::kVec; ++x) sums[warp][Joined<D>::dim(lane, c, x)] = j.acc[c][x];
        __syncthreads();
        if (warp != 0) return;
        for (int w = 0; w < kJoinWarps; ++w) j.m = fmaxf(j.m, sums[w][D]);
        const float base = j.m == -INFINITY ? 0.f : j.m;
        j.l = 0.f;
#pragma unroll
        for (int c = 0; c < Joined<D>::kParts; ++c)
#pragma unroll
            for (int x = 0; x < Joined<D>::kVec; ++x) j.acc[c][x] = 0.f;
        for (int w = 0; w < kJoinWarps; ++w) {
            const float weight = exp2_fast(sums[w][D] - base);
            j.l = fmaf(weight, sums[w][D + 1], j.l);
#pragma unroll
            for (int c = 0; c < Joined<D>::kParts; ++c)
#pragma unroll
                for (int x = 0; x < Joined<D>::kVec; ++x) j.acc[c][x] = fmaf(weight, sums[w][Joined<D>::dim(lane, c, x)], j.acc[c][x]);
        }
    } else if (warp != 0) {
        return;
    }
    j.template finish<T, TC>(p, h, n);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// One head's 16 rows of a page as [128-byte groups of columns][16 rows][128 bytes]
static bool group_map(const void* base, const fk_kv_cache& c, const int64_t* stride, CUtensorMap* out) {
    const int bytes = dtype_bytes(c.dtype), cols = 128 / bytes;
    const uint64_t dims[5] = {(uint64_t)cols, (uint64_t)c.page_size, (uint64_t)(c.head_dim / cols), (uint64_t)c.kv_heads, (uint64_t)c.pages};
    const uint64_t strides[4] = {(uint64_t)(stride[2] * bytes), 128, (uint64_t)(stride[1] * bytes), (uint64_t)(stride[0] * bytes)};
    const uint32_t box[5] = {(uint32_t)cols, (uint32_t)kFewKeys, (uint32_t)(c.head_dim / cols), 1, 1};
    return cache_tensor_map(base, c.dtype, 5, dims, strides, box, out);
}

template <int D, int NT, typename T, typename TC>
static int few(AttnParams p, int max_warps, size_t* need, cudaStream_t stream) {
    using S = FewShape<D, NT, TC>;
    p.tile_tokens = S::kCols / p.group;
    const int blocks = (int)min((int64_t)sm_count(), ((int64_t)max_warps + S::kWarps - 1) / S::kWarps);
    if (need) {
        *need = (size_t)blocks * 2 * (sizeof(PartHead) + (1 + S::kWarps) * S::kPart * sizeof(float));
        return FK_OK;
    }
    CUtensorMap key_map{}, value_map{};
    static std::atomic<uint64_t> allowed[2];
    auto launch = [&](auto kern, int tma) -> int {
        FK_CUDA_OK(allow_smem(kern, S::kSmem, allowed[tma]), "attention (few) attr");
        FK_CUDA_OK(launch_pdl(kern, dim3(blocks), dim3(32 * S::kWarps), (size_t)S::kSmem, stream, p, key_map, value_map), "attention (few) launch");
        FK_LAUNCH_OK("attention (few) launch");
        return FK_OK;
    };
    int st = -1;
    if constexpr (S::kPitch >= 128) {
        // Tensor copies where a group's rows lie in one page and its scales on 16 bytes: one instruction for what takes a warp 40 to 100
        auto scales_ok = [&](const float* s, const int64_t* stride) { return stride[2] == 1 && groups_aligned(s, stride, 2, 4, 16); };
        if (p.c.page_size % kFewKeys == 0 && (!S::kCodes || (scales_ok(p.c.key_scale, p.c.key_scale_stride) && scales_ok(p.c.value_scale, p.c.value_scale_stride))) &&
            group_map(p.c.key, p.c, p.c.key_stride, &key_map) && group_map(p.c.value, p.c, p.c.value_stride, &value_map))
            st = launch(attention_few_kernel<D, NT, T, TC, true>, 1);
    }
    if (st < 0) st = launch(attention_few_kernel<D, NT, T, TC, false>, 0);
    if (st != FK_OK) return st;
    const int cols = (int)min((int64_t)S::kCols, (int64_t)p.tile_tokens * p.group);
    FK_CUDA_OK(launch_pdl(attention_few_join_kernel<D, NT, T, TC>, dim3((unsigned)blocks, cols), dim3(32 * kJoinWarps), 0, stream, p), "attention (few) join launch");
    FK_LAUNCH_OK("attention (few) join launch");
    return FK_OK;
}

template <int D, typename T, typename TC>
static int few_columns(const AttnParams& p, int cols, int max_warps, size_t* need, cudaStream_t stream) {
    if constexpr (D < 256)
        if (cols > 8) return few<D, 2, T, TC>(p, max_warps, need, stream);
    return few<D, 1, T, TC>(p, max_warps, need, stream);
}

template <typename T, typename TC>
static int few_dim(const AttnParams& p, int cols, int max_warps, size_t* need, cudaStream_t stream) {
    switch (p.c.head_dim) {
        case 64: return few_columns<64, T, TC>(p, cols, max_warps, need, stream);
        case 128: return few_columns<128, T, TC>(p, cols, max_warps, need, stream);
        default: return few_columns<256, T, TC>(p, cols, max_warps, need, stream);
    }
}

bool attention_few_supported(const AttnParams& p, int dtype, int max_query) {
    if (dtype != FK_BF16 && dtype != FK_F16) return false;
    if (p.c.head_dim != 64 && p.c.head_dim != 128 && p.c.head_dim != 256) return false;
    // two groups of 8 columns do not fit the registers at 256 dimensions
    if (max_query < 1 || (int64_t)max_query * p.group > (p.c.head_dim == 256 ? 8 : 16)) return false;
    const int cb = dtype_bytes(p.c.dtype);
    return groups_aligned(p.c.key, p.c.key_stride, 3, cb, 16) && groups_aligned(p.c.value, p.c.value_stride, 3, cb, 16) && groups_aligned(p.query, p.qs, 2, 2, 4);
}

// need != null: only the workspace's size
int attention_few(const AttnParams& p, int dtype, int max_query, size_t* need, cudaStream_t stream) {
    // most runs that the call can have: no more warps are launched
    const int64_t longest = ((int64_t)p.c.max_pages * p.c.page_size + kFewKeys - 1) / kFewKeys;
    const int64_t groups = longest * p.c.kv_heads * (p.c.seqs < p.rows ? p.c.seqs : p.rows);
    const int max_warps = (int)min((int64_t)1 << 20, max((int64_t)1, (groups + kFewLeast - 1) / kFewLeast));
    const int cols = max_query * p.group;
    if (dtype == FK_BF16)
        return p.c.dtype == FK_E4M3 ? few_dim<__nv_bfloat16, __nv_fp8_e4m3>(p, cols, max_warps, need, stream)
                                    : few_dim<__nv_bfloat16, __nv_bfloat16>(p, cols, max_warps, need, stream);
    return p.c.dtype == FK_E4M3 ? few_dim<__half, __nv_fp8_e4m3>(p, cols, max_warps, need, stream) : few_dim<__half, __half>(p, cols, max_warps, need, stream);
}

}  // namespace fk
