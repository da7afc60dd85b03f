// Attention of chunks of new tokens over a paged cache on the tensor cores (tcgen05, two SMs per tile).
//
// A tile is 256 query rows (tokens x heads of the group) of one (sequence, key/value head) on a pair of SMs, 128 rows on each;
// it walks over its keys 128 at a time:
//   S[256, 128] = Q K^T          operands in shared memory, each SM holding 64 of the 128 keys
//   P = 2^(S - m)                two threads per row, 64 columns each, that exchange their maxima
//   O[256, dim] += P V           P from tensor memory, where it replaces S; each SM holds half of the values' columns
// The pair shares every key and value row, so an SM fetches half of them: at 256 dimensions one SM alone would need 64 bytes
// of L2 per clock for 128 rows, and the whole chip gets 41 (11.8 TB/s measured); a pair needs 32.  It is also what lets the ring
// hold 128-key tiles at 256 dimensions: 64 KB of queries + five slots of 32 KB.  Tensor memory: O (dim columns) and two S buffers
// (128 columns each), so the products of the next tile run while this tile's softmax is taken.
//
// Warps of a block: 0..7 softmax (and the scaling and storing of O), 8..11 producers (tensor copies out of the pages; where pages or
// strides do not allow them, and for codes, which become fp16 on the way, rows gathered by the threads), 12 issues the products (in
// the pair's first block), 13 zeroes value rows that nobody may see.  m is only raised when a row's maximum grows by more than
// 2^kLazy, which spares nearly all passes over O.  Weights are rounded to the type of the operands (fp16 after a factor 2^7, which with
// 2^kLazy stays below 2^15); sums are fp32.  Codes: a weight is multiplied by its value's scale before it is rounded, and by a power of two of
// the row's own, which follows the largest such product among the keys that the row sees: a scale far larger or smaller than the others,
// masked or of no weight, takes no bits from the rest.
//
// Key tiles of all tiles are dealt to the pairs in equal contiguous runs as in the few-row kernel; a run's first and last tile
// may be partial, and attention_tile_join_kernel joins those in key order.
//
// What bounds it (256 dimensions, 2048 tokens at 16384): a tile is 2050 clocks of products and 1030 of exponentials; the products of tile
// t + 1 need the S buffer that tile t - 1's weights leave, so a round is products + barrier + softmax of half a round, some 3100 clocks:
// 475 us, 1085 TFLOP/s, 0.66 of the measured cuBLAS rate (471 to 480 us from one machine to the next).

#include <cfloat>
#include <type_traits>

#include "attention_items.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace fk {

constexpr int kTileRows = 256, kTileKeys = 128;
constexpr int kTileThreads = 448;       // 14 warps of up to 128 registers
constexpr int kMetaRing = 8;
constexpr int kMmaWarp = 12, kEdgeWarp = 13;

template <int D, typename TC>
struct TileShape {
    static constexpr bool kCodes = sizeof(TC) == 1;
    static constexpr int kQuery = 128 * D * 2;                       // bytes of a block's query rows
    static constexpr int kSlot = 64 * D * 2;                         // 64 keys, or 128 values' half rows
    // Buffers of query rows.  With one, an item's first scores wait for the last products of the item before (its keys are then loaded
    // behind the other's last values); with two, items follow each other like the tiles of one
    static constexpr int kQueries = D == 256 ? 1 : 2;
    static constexpr int kSlots = D == 256 ? (kCodes ? 4 : 5) : (kCodes ? 8 : 9);
    static constexpr int kMeta = kMetaRing * (kCodes ? 3 * kTileKeys * 4 + 16 : 16);
    static constexpr int kExchange = (kCodes ? 2 : 1) * 2 * 2 * 128 * 4;      // between the two threads of a row
    static constexpr int kSmem = kQueries * kQuery + kSlots * kSlot + 640 + kMeta + kExchange + 4 * 128 * (kCodes ? 4 : 0);

    static constexpr int kPart = (D + 2) * kTileRows;                // floats of a partial result: m, l per row, [row][D]
    static_assert(kSmem <= 227 * 1024, "shared memory of a block");
    static_assert(2 * kMetaRing >= kSlots + 3, "a key tile's description outlives its softmax");
};

// A wait by parity only tells neighbouring phases apart.  s_full, p_full and o_done are waited for by warps that skip phases or come to
// them late, so each has one barrier for even and one for odd tiles: when tile t is waited for, t - 2 is known to be over and t + 2 cannot be.
struct TileBarriers {
    uint64_t full[12], empty[12], landed[12];
    uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2], o_empty;
    uint64_t keys_full[kMetaRing];
    uint32_t tmem;
    int abort_flag, odd, walked;
};
static_assert(sizeof(TileBarriers) <= 640, "fits behind the ring");

// ---- cluster-wide barriers and two-SM tensor-core instructions -----------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive at the barrier of the same offset in the pair's first block.  For what lies in tensor memory (ordered by the tcgen05 fences)
// and for byte counts; a release at cluster scope would wait for all of the thread's memory accesses, some 1300 clocks here, which
// doubled the time of a tile.
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
// The same behind this thread's (or, after __syncwarp, warp's) writes to shared memory, which the products of the pair read.
__device__ __forceinline__ void arrive_first_release(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* dst) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}
// Descriptors of operands in shared memory, 128-byte swizzle, 8-row (8-k) groups 1024 bytes apart: the low word (address, distance of
// 64-column groups for MN-major operands) moves, the high one is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t group) { return (addr >> 4) | ((group >> 4) << 16); }
// K-major a and b: rows of 64 elements (128 bytes)
__device__ __forceinline__ void pair_mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"((uint32_t)accumulate), "n"(kDescHigh) : "memory");
}
// a in tensor memory; b MN-major: 64 columns (128 bytes) per k
__device__ __forceinline__ void pair_mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b_low), "r"(idesc), "r"((uint32_t)accumulate), "n"(kDescHigh) : "memory");
}
__device__ __forceinline__ bool elect_lane() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// arrive at the barrier of this offset in both blocks when all products issued so far are done
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
template <typename OT>
__device__ __forceinline__ constexpr uint32_t pair_idesc(uint32_t n, bool b_mn_major) {
    constexpr uint32_t type = std::is_same<OT, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((256u >> 4) << 24);
}
// 32 consecutive 32-bit columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tile_copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float tile_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t tile_pack(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t tile_pack(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store32(void* p, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ uint4 codes8_to_half(uint2 c) {
    uint4 r;
    codes4_to_half(c.x, r.x, r.y);
    codes4_to_half(c.y, r.z, r.w);
    return r;
}

// Keys of a tile by column (and by value row): with tensor copies, column n is key n.  Where threads copy the rows, producer warp w looks
// up keys 32 w .. 32 w + 31 and puts 16 of them into each block's half of the columns: column n is key 32 (n % 64 / 16) + 16 (n / 64) + n % 16.

// Copies of a box of [unit rows][64 columns] out of one page into this block's shared memory, announced at the pair's first block's
// barrier (address in the cluster's window).
__device__ __forceinline__ void pair_tma_load(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(row), "r"(head), "r"(page)
        : "memory");
}
__device__ __forceinline__ uint32_t in_first_block(uint64_t* bar) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
    return a;
}
__device__ __forceinline__ void arrive_expect(uint32_t cluster_bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(cluster_bar), "r"(bytes) : "memory");
}

// Sets the flag at the same address of the pair's other block.
__device__ __forceinline__ void tell_other_block(int* flag) {
    asm volatile("{\n\t.reg .b32 a, r;\n\tmov.u32 r, %%cluster_ctarank;\n\txor.b32 r, r, 1;\n\tmapa.shared::cluster.u32 a, %0, r;\n\tst.shared::cluster.u32 [a], 1;\n\t}"
                 ::"r"(smem_u32(flag)) : "memory");
}

// Whether the cursor's key tile has keys that no row of the item sees.
__device__ __forceinline__ bool edge_tile(const AttnParams& p, const ItemCursor<kTileKeys>& c) {
    const int key0 = c.key0();
    return !(key0 + kTileKeys <= c.span.end && (p.window == 0 || key0 >= window_start(p, c.pos0) || key0 + kTileKeys <= p.sinks));
}

// Workspace: two parts' heads per pair, one mark per block (it wrote a whole item's row of several tokens that is not finite), the parts.
__host__ __device__ inline size_t tile_head_bytes(int pairs) { return (size_t)pairs * 2 * sizeof(PartHead) + ((size_t)pairs * 2 * sizeof(int) + 31) / 32 * 32; }
__device__ __forceinline__ int* tile_marks(const AttnParams& p, int pairs) { return reinterpret_cast<int*>(reinterpret_cast<PartHead*>(p.part) + 2 * pairs); }
__device__ __forceinline__ float* tile_parts(const AttnParams& p, int pairs) { return p.part + tile_head_bytes(pairs) / sizeof(float); }

// D: dimensions of the tiles, a multiple of 128 not below head_dim (the rest is zero).  T: type of queries and results, TC: of the
// cache.  TMA: rows come by tensor copies of `unit` rows (a divisor of the page size), else by the producers' threads.
template <int D, typename T, typename TC, bool TMA>
__global__ void __launch_bounds__(kTileThreads, 1) attention_tile_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap key_map,
                                                                         const __grid_constant__ CUtensorMap value_map, int unit) {
    static_assert(!TMA || sizeof(TC) == 2, "codes are converted by threads");
    using S = TileShape<D, TC>;
    constexpr bool kCodes = S::kCodes;
    using OT = typename std::conditional<kCodes, __half, TC>::type;
    constexpr bool kHalf = std::is_same<OT, __half>::value;
    constexpr float kShift = kHalf ? 7.f : 0.f, kUnshift = kHalf ? 0x1p-7f : 1.f;       // parts are kept without the weights' factor: large values
    constexpr float kLazy = 8.f - (kCodes ? 1.f : 0.f);
    constexpr int kSlots = S::kSlots;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + S::kQueries * S::kQuery;
    unsigned char* tail = smem + S::kQueries * S::kQuery + kSlots * S::kSlot;
    TileBarriers& bar = *reinterpret_cast<TileBarriers*>(tail);
    uint32_t* key_mask = reinterpret_cast<uint32_t*>(tail + 640);                       // [kMetaRing][4]
    float* key_scale = reinterpret_cast<float*>(tail + 640 + kMetaRing * 16);           // codes: [kMetaRing][128], by column
    float* value_scale = key_scale + kMetaRing * kTileKeys;                             // codes: [kMetaRing][128], by value row
    float* value_log = value_scale + kMetaRing * kTileKeys;                             // codes: the same, |value scale| < 2^this
    float* exchange = reinterpret_cast<float*>(tail + 640 + S::kMeta);                  // [2][2][128], codes: twice
    float* query_scale = exchange + S::kExchange / 4;                                   // codes: [4][128], by row of the block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) { mbar_init(&bar.full[i], 2); mbar_init(&bar.empty[i], 1); }
        for (int i = 0; i < kSlots; ++i) mbar_init(&bar.landed[i], TMA ? 1 : 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.q_full[i], 8);
            mbar_init(&bar.q_empty[i], 1);
            mbar_init(&bar.o_done[i], 1); mbar_init(&bar.s_full[i], 1); mbar_init(&bar.p_full[i], 16); }
        mbar_init(&bar.o_empty, 16);
        for (int i = 0; i < kMetaRing; ++i) mbar_init(&bar.keys_full[i], TMA ? 1 : 4);
        bar.abort_flag = bar.odd = bar.walked = 0;
        mbar_init_fence();
        if (TMA) {
            prefetch_tensormap(&key_map);
            prefetch_tensormap(&value_map);
        }
    }
    if (warp == kMmaWarp) pair_tmem_alloc(&bar.tmem);
    pdl_trigger();
    tc_fence_before_sync();
    cluster_sync();                                  // barriers are there in both blocks
    tc_fence_after_sync();
    const uint32_t tmem = bar.tmem, tmem_s = tmem + (D == 256 ? 256 : 128);
    volatile int* abort_flag = &bar.abort_flag;
    // Both blocks of the pair give up together: a warp whose wait fails issues nothing more, so whatever the other block then waits for
    // stays away, and what it has been given by then is right
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (warp_wait(b, parity, abort_flag, p.wait_cycles)) return true;
        bar.abort_flag = 1;
        tell_other_block(&bar.abort_flag);
        return false;
    };
    pdl_wait();

    int64_t* upto = reinterpret_cast<int64_t*>(smem);              // over the queries and the ring, before their first copy
    const int room = (S::kQueries * S::kQuery + kSlots * S::kSlot) / 8;
    const Runs runs{plan_tiles<kTileKeys>(p, reinterpret_cast<int64_t*>(exchange), upto, room), pairs, 1};
    const int64_t run0 = runs.begin(pair), run1 = runs.begin(pair + 1);
    const int tiles = (int)(run1 - run0);
    PartHead* heads = reinterpret_cast<PartHead*>(p.part) + 2 * (int64_t)pair;
    float* parts = tile_parts(p, pairs) + 2 * (int64_t)pair * S::kPart;
    if (threadIdx.x == 0 && rank == 0) heads[0].begins = heads[0].ends = heads[1].begins = heads[1].ends = -1;

    ItemCursor<kTileKeys> c;
    if (tiles > 0) locate(p, run0, upto, room, c);
    fence_async_proxy();                             // the plan's memory is the copies' from here on
    __syncthreads();
    if (tiles > 0) {
        const int dim = p.c.head_dim;
        if (warp >= 8 && warp < kMmaWarp) {
            // ------------------------------------------------------------------------------------------------- producers
            const int w = warp - 8;
            int page = -1, in_page = 0;              // of key w * 32 + lane of the cursor's tile
            auto look = [&] {
                page = -1;
                const int j = c.key0() + w * 32 + lane;
                if (c.some_row_sees(p, j)) page = page_of(p.c, c.seq, j, in_page);
            };
            int x = 0;                               // loads so far
            bool alive = true;                       // no wait has failed
            int arrived = 0;                         // of them announced
            constexpr int kLag = 2;                  // loads in flight behind the newest
            auto announce = [&](int upto) {          // loads below `upto` have landed for this thread
                fence_async_proxy();
                __syncwarp();
                for (; arrived < upto; ++arrived)
                    if (lane == 0) mbar_arrive(&bar.landed[arrived % kSlots]);
            };
            // Whether the next load's slot is free, the same for all lanes: one that sees the phase change before another must not leave the
            // warp alone in what follows, which announces loads for all of it
            auto slot_free = [&] { return __all_sync(kFull, mbar_try_wait(&bar.empty[x % kSlots], ((x / kSlots) & 1) ^ 1)) != 0; };
            auto wait_slot = [&] { return wait(&bar.empty[x % kSlots], ((x / kSlots) & 1) ^ 1); };
            auto load_query = [&](int segment) {     // 32 of the block's 128 rows per warp
                if (!kCodes && !TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
                if (!TMA) announce(x);               // the products that read the old rows wait for these loads
                const int cols = c.tokens(p) * p.group, first_row = c.first_row(p);
                constexpr int kChunks = D / 8, kAtOnce = 32 / kChunks < 1 ? 1 : 32 / kChunks, kSteps = 32 / kAtOnce, kBatch = 8;
                const int chunk = lane % kChunks;
                const int buffer = segment % S::kQueries;
                const uint32_t to = q_smem + buffer * S::kQuery + (chunk >> 3) * (128 * 128);
                auto source = [&](int r) -> const T* {           // null: padding
                    const int n = rank * 128 + r, tok = n / p.group;
                    if (n >= cols || chunk * 8 >= dim) return nullptr;
                    return reinterpret_cast<const T*>(p.query) + (int64_t)(first_row + tok) * p.qs[0] + (int64_t)(c.head * p.group + n - tok * p.group) * p.qs[1] + chunk * 8;
                };
                auto free_buffer = [&] { return wait(&bar.q_empty[buffer], ((segment / S::kQueries) & 1) ^ 1); };
                if (!kCodes) {
                    if (!(alive = free_buffer())) return;
#pragma unroll 4
                    for (int i = 0; i < kSteps; ++i) {
                        const int r = w * 32 + i * kAtOnce + lane / kChunks;
                        const T* q = source(r);
                        tile_copy16(to + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), q ? q : p.query, q ? 16 : 0);
                    }
                    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                } else {
                    for (int i0 = 0; i0 < kSteps; i0 += kBatch) {
                        uint4 raw[kBatch];
#pragma unroll
                        for (int b = 0; b < kBatch; ++b) {
                            const T* q = source(w * 32 + (i0 + b) * kAtOnce + lane / kChunks);
                            raw[b] = q ? *reinterpret_cast<const uint4*>(q) : make_uint4(0, 0, 0, 0);
                        }
                        if (i0 == 0 && !(alive = free_buffer())) return;
#pragma unroll
                        for (int b = 0; b < kBatch; ++b) {
                            const int r = w * 32 + (i0 + b) * kAtOnce + lane / kChunks;
                            float v[8], most = 0.f;
                            load8<true>(reinterpret_cast<const T*>(&raw[b]), 8, v);
#pragma unroll
                            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
#pragma unroll
                            for (int o = kChunks / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, o));
                            const int e2 = row_exponent(most);
                            const float down = ldexpf(1.f, -e2);
                            uint4 out;
                            uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[e] = tile_pack(v[2 * e] * down, v[2 * e + 1] * down, OT{});
                            if (chunk == 0) query_scale[(segment & 3) * 128 + r] = fmaxf(ldexpf(fabsf(p.scale_log2), e2), FLT_MIN);
                            sts16(to + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), out);
                        }
                    }
                }
                fence_async_proxy();
                __syncwarp();
                if (lane == 0) arrive_first_release(&bar.q_full[buffer]);
            };
            // rows of a slot: keys take 16 of this warp's 32 (those of this block's half), values all 32 with half of their columns
            constexpr int kKeyChunks = D / 8, kKeyAtOnce = 32 / kKeyChunks < 1 ? 1 : 32 / kKeyChunks;
            constexpr int kValueChunks = D / 16, kValueAtOnce = 32 / kValueChunks;
            auto key_addr = [&](uint32_t base, int i, int chunk) {
                const int r = w * 16 + i;
                return base + (chunk >> 3) * (64 * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
            };
            auto value_addr = [&](uint32_t base, int i, int chunk) {
                const int r = (i >> 4) * 64 + w * 16 + (i & 15);
                return base + (chunk >> 3) * (128 * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
            };
            // threads' copies of 16-bit rows; offset: bytes of this lane's row, < 0: no such row
            auto load = [&](bool values, int64_t offset) {
                const int slot = x % kSlots;
                if (!slot_free()) {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");      // ahead of the products: announce what is on its way first
                    announce(x);
                    if (!(alive = wait_slot())) return;
                }
                const uint32_t base = ring + slot * S::kSlot;
                const char* from = reinterpret_cast<const char*>(values ? p.c.value : p.c.key);
                if (!values) {
#pragma unroll
                    for (int i0 = 0; i0 < 16; i0 += kKeyAtOnce) {
                        const int i = i0 + lane / kKeyChunks, chunk = lane % kKeyChunks;
                        const int64_t off = __shfl_sync(kFull, offset, rank * 16 + i);
                        const bool there = off >= 0 && chunk * 8 < dim;
                        tile_copy16(key_addr(base, i, chunk), there ? from + off + chunk * 16 : from, there ? 16 : 0);
                    }
                } else {
#pragma unroll
                    for (int i0 = 0; i0 < 32; i0 += kValueAtOnce) {
                        const int i = i0 + lane / kValueChunks, chunk = lane % kValueChunks, at = rank * kValueChunks + chunk;
                        const int64_t off = __shfl_sync(kFull, offset, i);
                        const bool there = off >= 0 && at * 8 < dim;
                        tile_copy16(value_addr(base, i, chunk), there ? from + off + at * 16 : from, there ? 16 : 0);
                    }
                }
                ++x;
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (x > kLag) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                    announce(x - kLag);
                }
            };
            // codes: all of a thread's reads of a slot at once, converted and stored when the slot is free
            constexpr int kRaw = 16 / kKeyAtOnce;                // pieces of eight codes per thread, of keys as of values
            static_assert(kRaw == 32 / kValueAtOnce, "half of the keys, half of the values' columns");
            auto fetch = [&](bool values, int64_t offset, uint2 (&raw)[kRaw]) {
                const char* from = reinterpret_cast<const char*>(values ? p.c.value : p.c.key);
#pragma unroll
                for (int r = 0; r < kRaw; ++r) {
                    const int i = values ? r * kValueAtOnce + lane / kValueChunks : rank * 16 + r * kKeyAtOnce + lane / kKeyChunks;
                    const int chunk = values ? rank * kValueChunks + lane % kValueChunks : lane % kKeyChunks;
                    const int64_t off = __shfl_sync(kFull, offset, i);
                    raw[r] = off >= 0 && chunk * 8 < dim ? *reinterpret_cast<const uint2*>(from + off + chunk * 8) : make_uint2(0, 0);
                }
            };
            auto put = [&](bool values, int64_t offset) {
                uint2 raw[kRaw];
                fetch(values, offset, raw);
                const int slot = x % kSlots;
                if (!(alive = wait_slot())) return;
                const uint32_t base = ring + slot * S::kSlot;
#pragma unroll
                for (int r = 0; r < kRaw; ++r)
                    sts16(values ? value_addr(base, r * kValueAtOnce + lane / kValueChunks, lane % kValueChunks) : key_addr(base, r * kKeyAtOnce + lane / kKeyChunks, lane % kKeyChunks),
                          codes8_to_half(raw[r]));
                ++x;
                announce(x);
            };
            int segment = 0;
            bool first = true;
            if (TMA) {
                    // A copy takes its warp some 130 clocks to issue, so the four warps take every fourth one each
                    const int units = kTileKeys / unit, key_units = units / 2;
                    // lane i < units: unit i of the cursor's tile; its page, -1 where the table holds none, -2 where no row sees the unit.
                    // Copies of no page are from behind the last one, which reads as zeros
                    int page = 0, row = 0, page_v = 0, row_v = 0, head_v = 0;
                    bool edge_v = false;
                    auto look_unit = [&] {
                        page = -2;
                        const int j = c.key0() + lane * unit;
                        if (lane < units && j < c.span.end && (p.window == 0 || j + unit > window_start(p, c.pos0) || j < p.sinks)) page = page_of(p.c, c.seq, j, row);
                    };
                    auto tma_values = [&] {
                        constexpr int groups = D / 128;
                        const int slot = x % kSlots;
                        if (!(alive = wait_slot())) return;
                        uint32_t to = in_first_block(&bar.full[slot]);
                        if (edge_v) to = smem_u32(&bar.landed[slot]);
                        if (lane == 0 && w == 0) {
                            if (edge_v) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(to), "r"((uint32_t)S::kSlot) : "memory");
                            else arrive_expect(to, S::kSlot);
                        }
                        __syncwarp();
                        const int u = lane / groups, g = lane % groups;
                        const int pg = __shfl_sync(kFull, page_v, u), rw = __shfl_sync(kFull, row_v, u);
                        if (u < units && (lane & 3) == w)
                            pair_tma_load(ring + slot * S::kSlot + g * (128 * 128) + u * unit * 128, &value_map, (rank * groups + g) * 64, rw, head_v, pg < 0 ? p.c.pages : pg, to);
                        ++x;
                    };
                    look_unit();
                    for (int t = 0; t < tiles; ++t) {
                        constexpr int groups = D / 64;
                        if (S::kQueries == 1 && first && t > 0) tma_values();
                        if (!alive) break;
                        const int slot = x % kSlots, meta = t % kMetaRing, head = c.head;
                        const bool edge = edge_tile(p, c), ends = c.k + 1 >= c.span.count, values_now = t > 0 && !(S::kQueries == 1 && first);
                        if (!(alive = wait_slot())) break;       // and with it for the last reader of this description (static_assert above)
                        const uint32_t full = in_first_block(&bar.full[slot]);
                        const unsigned there = __ballot_sync(kFull, page != -1) & (0xffffffffu >> (32 - units));
                        if (lane == 0 && w == 0) {
                            key_mask[meta * 4] = there;          // one bit per unit: not missing
                            mbar_arrive(&bar.keys_full[meta]);
                            arrive_expect(full, S::kSlot);
                            *reinterpret_cast<volatile int*>(&bar.walked) = t;
                        }
                        __syncwarp();
                        const int u = lane / groups, g = lane % groups;
                        const int pg = __shfl_sync(kFull, page, (rank * key_units + u) & 31), rw = __shfl_sync(kFull, row, (rank * key_units + u) & 31);
                        if (u < key_units && (lane & 3) == w)
                            pair_tma_load(ring + slot * S::kSlot + g * (64 * 128) + u * unit * 128, &key_map, g * 64, rw, head, pg < 0 ? p.c.pages : pg, full);
                        ++x;
                        if (first) load_query(segment);
                        if (!alive) break;
                        // on to the next tile: its page numbers arrive while the previous tile's values are issued
                        const int page_now = page, row_now = row;
                        if (t + 1 < tiles) {
                            if (ends) c.next_item(p); else ++c.k;
                            look_unit();
                        }
                        if (values_now) tma_values();
                        if (!alive) break;
                        page_v = page_now; row_v = row_now; head_v = head; edge_v = edge;
                        first = ends;
                        if (ends) ++segment;
                    }
                    if (alive) tma_values();
            }
            if (!TMA) {
                int64_t key_offset = -1, value_offset = -1, next_value = -1;         // of the tile at hand, of the one before, of the tile at hand
                float ks = 0.f, vs = 0.f;
                auto place = [&] {                   // of the cursor's tile, looked up before
                    key_offset = page < 0 ? -1 : row_offset(p.c.key_stride, page, c.head, in_page) * (int64_t)sizeof(TC);
                    next_value = page < 0 ? -1 : row_offset(p.c.value_stride, page, c.head, in_page) * (int64_t)sizeof(TC);
                    if constexpr (kCodes) {
                        ks = page < 0 ? 0.f : p.c.key_scale[row_offset(p.c.key_scale_stride, page, c.head, in_page)];
                        vs = page < 0 ? 0.f : p.c.value_scale[row_offset(p.c.value_scale_stride, page, c.head, in_page)];
                    }
                };
                auto store_values = [&] {
                    if constexpr (kCodes) put(true, value_offset); else load(true, value_offset);
                };
                look();
                place();
                for (int t = 0; t < tiles; ++t) {
                    if (first) {
                        if (S::kQueries == 1 && t > 0) store_values();
                        if (alive) load_query(segment);
                    }
                    if (!alive) break;
                    // this tile's rows: which of them are there, their scales.  A description is written anew only when its last reader has
                    // passed: the key slot of this tile was freed later than that (static_assert above); so wait for the slot first
                    const unsigned rows = __ballot_sync(kFull, page >= 0);
                    const int meta = t % kMetaRing;
                    if (!slot_free()) {
                        if (!kCodes) {
                            asm volatile("cp.async.wait_group 0;" ::: "memory");
                            announce(x);
                        }
                        if (!(alive = wait_slot())) break;
                    }
                    if (lane == 0) key_mask[meta * 4 + w] = rows;
                    if (kCodes) {
                        const int n = (lane >> 4) * 64 + w * 16 + (lane & 15);
                        key_scale[meta * kTileKeys + n] = ks;
                        value_scale[meta * kTileKeys + n] = vs;
                        value_log[meta * kTileKeys + n] = vs == 0.f ? -INFINITY : (float)((int)((__float_as_uint(vs) >> 23) & 255) - 126);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar.keys_full[meta]);
                    // on to the next tile before the copies: its page numbers arrive meanwhile
                    const bool ends = c.k + 1 >= c.span.count;
                    const int64_t value_now = next_value;
                    const bool more = t + 1 < tiles;
                    if (more) {
                        if (ends) c.next_item(p); else ++c.k;
                        look();
                    }
                    if constexpr (kCodes) put(false, key_offset); else load(false, key_offset);
                    if (alive && t > 0 && !(S::kQueries == 1 && first)) store_values();
                    if (!alive) break;
                    value_offset = value_now;
                    if (more) place();
                    first = ends;
                    if (ends) ++segment;
                }
                if (alive) store_values();
                if (!kCodes) {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    announce(x);
                }
            }
            // The products' last arrivals at this block's barriers, which nobody else waits for: the block must still be there
            if (w == 0 && alive) {
                for (int i = max(0, x - kSlots); i < x && alive; ++i) alive = wait(&bar.empty[i % kSlots], (i / kSlots) & 1);
                const int queries = first ? segment : segment + 1;
                for (int i = max(0, queries - S::kQueries); i < queries && alive; ++i) alive = wait(&bar.q_empty[i % S::kQueries], (i / S::kQueries) & 1);
            }
        } else if (warp == kEdgeWarp) {
            // ------------------------------------------------------------------------------------------------- edges
            // A tile of values with rows that nobody may see (behind the sequence's end, outside of the window) is copied to a barrier of
            // its own: here those rows are zeroed, which can hold anything (0 * infinity is no zero), and the slot is announced.
            if (TMA) {
                uint32_t landed = 0;                     // per slot: parity of its next such copy
                // From one such tile to the next may be an item's whole time: the limit counts from the producers' last tile
                auto wait_long = [&](uint64_t* b, uint32_t parity) {
                    while (true) {
                        const int walked = __shfl_sync(kFull, *reinterpret_cast<volatile int*>(&bar.walked), 0);
                        if (warp_wait(b, parity, abort_flag, p.wait_cycles)) return true;
                        if (__any_sync(kFull, *abort_flag != 0 || *reinterpret_cast<volatile int*>(&bar.walked) == walked)) return wait(b, parity);
                    }
                };
                for (int t = 0; t < tiles; ++t) {
                    const bool ends = c.k + 1 >= c.span.count;
                    if (edge_tile(p, c)) {
                        // order of the loads: K(0), then [K(t + 1), V(t)], but [V(t), K(t + 1)] where t ends an item and there is one query buffer
                        const int slot = ((S::kQueries == 1 && ends) || t + 1 == tiles ? 2 * t + 1 : 2 * t + 2) % kSlots, key0 = c.key0(), lo = window_start(p, c.pos0);
                        const uint32_t base = ring + slot * S::kSlot;
                        if (!wait_long(&bar.landed[slot], (landed >> slot) & 1)) break;
                        landed ^= 1u << slot;
                        for (int r = lane; r < kTileKeys; r += 32) {
                            const int j = key0 + r;
                            if (j < c.span.end && (p.window == 0 || j >= lo || j < p.sinks)) continue;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) sts16(base + (i >> 3) * (128 * 128) + r * 128 + ((i & 7) << 4), make_uint4(0, 0, 0, 0));
                        }
                        fence_async_proxy();
                        __syncwarp();
                        if (lane == 0) arrive_first_release(&bar.full[slot]);
                    }
                    if (t + 1 < tiles) {
                        if (ends) c.next_item(p); else ++c.k;
                    }
                }
            } else {
                // rows written by the producers' threads: announced to the pair from here, because a release at cluster scope waits for all
                // of its thread's memory accesses, and this warp has none
                for (int x = 0; x < 2 * tiles; ++x) {
                    if (!wait(&bar.landed[x % kSlots], (x / kSlots) & 1)) break;
                    if (lane == 0) arrive_first_release(&bar.full[x % kSlots]);
                    __syncwarp();
                }
            }
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------------------------------------------------- products
            // The whole warp walks and waits, one lane issues: what the instructions need is then the same for all lanes and lies in uniform
            // registers, and the issuing thread's own instructions are not what bounds a tile (with all of it in one lane's branch, a tile
            // took 4000 clocks for 2050 of products)
            if (rank == 0) {
                constexpr uint32_t s_idesc = pair_idesc<OT>(kTileKeys, false), o_idesc = pair_idesc<OT>(D, true);
                const uint32_t q_low = desc_low(q_smem, 16), k_low = desc_low(ring, 16), v_low = desc_low(ring, 128 * 128);
                const bool leader = elect_lane();
                int slot = 0, segment = 0, o_segment = 0;
                uint32_t phase = 0;                  // of the ring
                auto next = [&] {
                    if (++slot == kSlots) { slot = 0; phase ^= 1; }
                };
                auto scores = [&](int t, bool ends, int buffer) {
                    if (!wait(&bar.full[slot], phase)) return false;
                    tc_fence_after_sync();
                    if (leader) {
                        const uint32_t d = tmem_s + (t & 1) * kTileKeys, k = k_low + slot * (S::kSlot >> 4), q = q_low + buffer * (S::kQuery >> 4);
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
                            if (i * 16 < dim) pair_mma_ss(d, q + (((i >> 2) * (128 * 128) + (i & 3) * 32) >> 4), k + (((i >> 2) * (64 * 128) + (i & 3) * 32) >> 4), s_idesc, i > 0);
                        pair_commit(&bar.s_full[t & 1]);
                        pair_commit(&bar.empty[slot]);
                        if (ends) pair_commit(&bar.q_empty[buffer]);
                    }
                    __syncwarp();
                    next();
                    return true;
                };
                auto values = [&](int t, bool begins) {
                    if (!wait(&bar.full[slot], phase)) return false;
                    if (begins) {
                        if (o_segment > 0 && !wait(&bar.o_empty, (o_segment - 1) & 1)) return false;
                        ++o_segment;
                    }
                    if (!wait(&bar.p_full[t & 1], (t >> 1) & 1)) return false;
                    tc_fence_after_sync();
                    if (leader) {
                        const uint32_t a = tmem_s + (t & 1) * kTileKeys, v = v_low + slot * (S::kSlot >> 4);
#pragma unroll
                        for (int i = 0; i < kTileKeys / 16; ++i) pair_mma_ts(tmem, a + i * 8, v + i * (2048 >> 4), o_idesc, !begins || i > 0);
                        pair_commit(&bar.o_done[t & 1]);
                        pair_commit(&bar.empty[slot]);
                    }
                    __syncwarp();
                    next();
                    return true;
                };
                bool first = true, last_began = false, alive = true;
                for (int t = 0; t < tiles; ++t) {
                    const bool ends = c.k + 1 >= c.span.count;
                    if (first) {
                        if (S::kQueries == 1 && t > 0) alive = values(t - 1, last_began);
                        alive = alive && wait(&bar.q_full[segment % S::kQueries], (segment / S::kQueries) & 1);
                        ++segment;
                    }
                    alive = alive && scores(t, ends || t + 1 == tiles, (segment - 1) % S::kQueries);
                    if (t > 0 && !(S::kQueries == 1 && first)) alive = alive && values(t - 1, last_began);
                    if (!alive) break;
                    last_began = first;
                    first = ends;
                    if (t + 1 < tiles) {
                        if (ends) c.next_item(p); else ++c.k;
                    }
                }
                if (alive) values(tiles - 1, last_began);
            }
        } else {
            // ------------------------------------------------------------------------------------------------- softmax
            // two threads per row, 64 columns each: warps w and w + 4
            const int quarter = warp & 3, half = warp >> 2;
            const int r = quarter * 32 + lane, n = rank * 128 + r;       // row of the block, of the pair
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            const uint32_t o_addr = tmem + lanes;
            float m = -INFINITY, l = 0.f, qscale = fabsf(p.scale_log2);
            // codes: the largest log2 of weight x value scale met so far, and the power of two (less m) that such products are held by
            float m_out = -INFINITY, k_out = 0.f;
            auto pow2 = [](float k) { return __int_as_float((127 + (int)k) << 23); };
            bool begins = true;                                          // of this run's part of the item
            // When a wait fails the walk goes on without waiting or announcing (the two warps of a row still meet), and every sum from
            // here on is no number: the factor of the scores says so, which takes no register
            auto dead = [&] { return qscale != qscale; };
            auto wait_or_die = [&](uint64_t* b, uint32_t parity) {
                if (!wait(b, parity)) qscale = NAN;
            };
            int segment = 0;
            int64_t at = run0;                                           // tile of the order
            int began_k = c.k;
            const int tok = n / p.group;
            const bool negative = p.scale_log2 < 0.f;
            auto meet = [&] { named_bar_sync(1 + quarter, 64); };
            for (int t = 0; t < tiles; ++t, ++at) {
                const int pos = c.pos0 + tok, meta = t % kMetaRing;
                const int key0 = c.key0();
                const bool inside = key0 + kTileKeys - 1 <= c.pos0 && (p.window == 0 || key0 >= window_start(p, c.pos1) || key0 + kTileKeys <= p.sinks);
                wait_or_die(&bar.keys_full[meta], (t / kMetaRing) & 1);
                uint32_t there[2] = {0xffffffffu, 0xffffffffu};          // one bit per key: its page is not missing
                bool complete;
                if (TMA) {
                    const uint32_t bits = key_mask[meta * 4];
                    complete = bits == 0xffffffffu >> (32 - kTileKeys / unit);
                    if (!complete)
                        for (int k = 0; k < 64; ++k)
                            if (!((bits >> ((half * 64 + k) / unit)) & 1u)) there[k >> 5] &= ~(1u << (k & 31));
                } else {
                    const uint4 v = *reinterpret_cast<const uint4*>(key_mask + meta * 4);
                    complete = (v.x & v.y & v.z & v.w) == 0xffffffffu;
                    // columns 16 i .. 16 i + 15 of this half are the half's 16 keys of producer warp i
                    there[0] = ((v.x >> (16 * half)) & 0xffffu) | ((v.y >> (16 * half)) << 16);
                    there[1] = ((v.z >> (16 * half)) & 0xffffu) | ((v.w >> (16 * half)) << 16);
                }
                wait_or_die(&bar.s_full[t & 1], (t >> 1) & 1);
                tc_fence_after_sync();
                const uint32_t s_addr = tmem_s + lanes + (t & 1) * kTileKeys;
                float s[64];
                tmem_ld32(s_addr + half * 64, s);
                tmem_ld32(s_addr + half * 64 + 32, s + 32);
                tmem_wait_ld();
                if (begins) {
                    m = -INFINITY;
                    l = 0.f;
                    m_out = -INFINITY;
                    k_out = 0.f;
                    if (kCodes && !dead()) qscale = query_scale[(segment & 3) * 128 + r];
                    began_k = c.k;
                }
                if (kCodes) {
                    const float4* ks = reinterpret_cast<const float4*>(key_scale + meta * kTileKeys + half * 64);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 f = ks[i];
                        s[4 * i] *= f.x; s[4 * i + 1] *= f.y; s[4 * i + 2] *= f.z; s[4 * i + 3] *= f.w;
                    }
                }
                if (negative)
#pragma unroll
                    for (int i = 0; i < 64; ++i) s[i] = -s[i];
                if (!complete || !inside) {
                    // column i of this half is key i (tensor copies), or 32 (i / 16) + i % 16 of those from 16 half on
                    uint32_t bits[2];
                    if (TMA) {
                        bits[0] = seen_bits(p, pos, key0 + half * 64);
                        bits[1] = seen_bits(p, pos, key0 + half * 64 + 32);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            bits[i] = (seen_bits(p, pos, key0 + 64 * i + 16 * half) & 0xffffu) | (seen_bits(p, pos, key0 + 64 * i + 32 + 16 * half) << 16);
                    }
                    bits[0] &= there[0];
                    bits[1] &= there[1];
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!((bits[i >> 5] >> (i & 31)) & 1u)) s[i] = -INFINITY;
                }
                // ---- the row's maximum; the base of the powers only moves when it has to
                float tops[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) tops[e] = fmaxf(s[e], s[e + 8]);
#pragma unroll
                for (int i = 16; i < 64; i += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) tops[e] = fmaxf(tops[e], fmaxf(s[i + e], s[i + 8 + e]));
                float most = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
                float* ex = exchange + (t & 1) * 256;
                ex[half * 128 + r] = most;
                float most_out = -INFINITY;
                if (kCodes) {
                    const float4* vl = reinterpret_cast<const float4*>(value_log + meta * kTileKeys + half * 64);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 f = vl[i];
                        most_out = fmaxf(most_out, fmaxf(fmaxf(fmaf(s[4 * i], qscale, f.x), fmaf(s[4 * i + 1], qscale, f.y)),
                                                         fmaxf(fmaf(s[4 * i + 2], qscale, f.z), fmaf(s[4 * i + 3], qscale, f.w))));
                    }
                    ex[512 + half * 128 + r] = most_out;
                }
                meet();                                                  // also: both have read their scores
                most = qscale * fmaxf(most, ex[(half ^ 1) * 128 + r]);
                float alpha = 1.f;
                const float m_new = most > m + kLazy ? most : m;
                const bool raised = m_new > m;
                const float fell = m - m_new;                            // log2 of what the older weights are worth now
                if (raised) alpha = m == -INFINITY ? 0.f : tile_exp2(fell);
                m = m_new;
                float factor = alpha;
                if (kCodes) {
                    const bool none = m_out == -INFINITY;                // no product but zeros so far
                    m_out = fmaxf(m_out, fmaxf(most_out, ex[512 + (half ^ 1) * 128 + r]));
                    // kept within 2^kLazy of the largest product; p 2^-k_out below stays finite
                    if (m_out > -INFINITY && (raised || none || m_out - m > k_out + kLazy)) {
                        const float k = fminf(fmaxf(ceilf(m_out - m), -112.f), 112.f);
                        if (alpha != 0.f) factor = tile_exp2((raised ? fell : 0.f) + k_out - k);
                        k_out = k;
                    }
                }
                if (!begins) {
                    if (__any_sync(kFull, factor != 1.f)) {              // the same in both warps of a row
                        wait_or_die(&bar.o_done[(t - 1) & 1], ((t - 1) >> 1) & 1);
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int i = half * (D / 2); i < (half + 1) * (D / 2); i += 16) {
                            float o[16];
                            tmem_ld16(o_addr + i, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= factor;
                            tmem_st16(o_addr + i, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                    l *= alpha;
                }
                // ---- weights
                const float base = m == -INFINITY ? 0.f : m - kShift;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                const float down_out = kCodes ? pow2(-k_out) : 1.f;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = part * 32 + 2 * i;
                        float a = tile_exp2(fmaf(s[e], qscale, -base)), b = tile_exp2(fmaf(s[e + 1], qscale, -base));
                        sum[i & 3] += a + b;
                        if (kCodes) {
                            const float2 vs = *reinterpret_cast<const float2*>(value_scale + meta * kTileKeys + half * 64 + e);
                            a = (a * down_out) * vs.x;                   // in this order: a weight of zero stays zero beside any scale
                            b = (b * down_out) * vs.y;
                        }
                        w[i] = tile_pack(a, b, OT{});
                    }
                    tmem_st16(s_addr + half * 32 + part * 16, w);        // over scores that both threads have read
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0 && !dead()) arrive_first(&bar.p_full[t & 1]);
                // ---- the end of the item, or of the run
                const bool ends = c.k + 1 >= c.span.count;
                if (ends || t + 1 == tiles) {
                    // the row's sum; the buffer is the one that the next tile's maxima do not use
                    float* sums = exchange + ((t + 1) & 1) * 256;
                    sums[half * 128 + r] = l;
                    meet();
                    l = sums[r] + sums[128 + r];                         // in this order in both threads
                    if (t > 0) wait_or_die(&bar.o_done[(t - 1) & 1], ((t - 1) >> 1) & 1);      // long over; at the run's end nobody else sees that it arrived
                    wait_or_die(&bar.o_done[t & 1], (t >> 1) & 1);
                    tc_fence_after_sync();
                    const int tokens = c.tokens(p), cols = tokens * p.group, first_row = c.first_row(p);
                    const bool whole = ends && began_k == 0;
                    if (dead()) l = NAN;
                    const float scale_out = dead() ? NAN : kCodes ? pow2(k_out) : 1.f;
                    const int which = at - (c.k - began_k) == run0 ? 0 : 1;
                    float* part = parts + which * (int64_t)S::kPart;
                    T* out = reinterpret_cast<T*>(p.out) + (int64_t)(first_row + tok) * p.os[0] + (int64_t)(c.head * p.group + n - tok * p.group) * p.os[1];
                    const float inv = l == 0.f ? 0.f : scale_out / l;
                    bool odd = false;
                    const bool wide = (dim & 15) == 0 && ((p.os[0] | p.os[1]) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
#pragma unroll 1
                    for (int i = half * (D / 2); i < (half + 1) * (D / 2); i += 16) {
                        float o[16];
                        tmem_ld16(o_addr + i, o);
                        if (n < cols && i < dim) {
                            if (whole) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    o[e] = l == 0.f ? 0.f : o[e] * inv;
                                    if (i + e < dim) odd |= !(fabsf(o[e]) < INFINITY);
                                }
                                // a row per thread: 32 bytes at a time fill whole sectors
                                if (wide) {
                                    uint32_t w[8];
#pragma unroll
                                    for (int e = 0; e < 8; ++e) w[e] = tile_pack(o[2 * e], o[2 * e + 1], T{});
                                    store32(out + i, w);
                                } else {
#pragma unroll
                                    for (int e = 0; e < 16; ++e)
                                        if (i + e < dim) store_elem(out + i + e, o[e]);
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= scale_out * kUnshift;
                                store32(part + 2 * kTileRows + (int64_t)n * D + i, reinterpret_cast<const uint32_t*>(o));
                                store32(part + 2 * kTileRows + (int64_t)n * D + i + 8, reinterpret_cast<const uint32_t*>(o + 8));
                            }
                        }
                    }
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0 && !dead()) arrive_first(&bar.o_empty);
                    if (whole) {
                        // the join kernel sees to rows whose result is not finite: nothing here waits for that
                        if (odd && l == l && tokens > 1) bar.odd = 1;
                    } else {
                        if (n < cols && half == 0) { part[n] = m; part[kTileRows + n] = l * kUnshift; }
                        if (rank == 0 && threadIdx.x == 0)
                            heads[which] = PartHead{first_row, tokens, c.head, c.seq, c.pos0, began_k == 0, ends, runs.worker_of(at - c.k + c.span.count - 1)};
                    }
                    ++segment;
                    meet();                                              // the exchange is free again
                }
                begins = ends;
                if (t + 1 < tiles) {
                    if (ends) c.next_item(p); else ++c.k;
                }
            }
        }
    }
    if (*abort_flag) linger();                       // copies and products still on their way to either block
    __syncwarp();
    tc_fence_before_sync();
    cluster_sync();                                  // nothing more arrives at either block's barriers
    if (threadIdx.x == 0) tile_marks(p, pairs)[blockIdx.x] = bar.odd;
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        pair_tmem_dealloc(tmem);
    }
}

// Rows of the whole items of this block's pair that are not finite (row_again): the pair's run is walked once more, its rows dealt to the warps
// of the blocks of the same pair.
template <typename T, typename TC>
__device__ __noinline__ void odd_rows_of_run(const AttnParams& p) {
    __shared__ int64_t scratch[2 * 8];
    const Runs runs{plan_tiles<kTileKeys>(p, scratch, nullptr, 0), (int64_t)gridDim.x, 1};
    const int64_t run1 = runs.begin(blockIdx.x + 1);
    int64_t at = runs.begin(blockIdx.x);
    ItemCursor<kTileKeys> c;
    locate(p, at, nullptr, 0, c);
    while (at < run1) {
        const int steps = (int)min((int64_t)(c.span.count - c.k), run1 - at), tokens = c.tokens(p);
        if (c.k == 0 && steps == c.span.count && tokens > 1)
            for (int n = blockIdx.y * 8 + (threadIdx.x >> 5); n < tokens * p.group; n += gridDim.y * 8)
                row_again<T, TC>(p, c.seq, c.first_row(p), c.pos0, tokens, n / p.group, c.head * p.group + n % p.group);
        at += steps;
        if (at < run1) c.next_item(p);
    }
}

// Joins the parts of one tile: block (pair whose run has the tile's beginning, 32 rows), four rows per warp, four dimensions per lane.
template <int D, typename T, typename TC>
__global__ void __launch_bounds__(256, 4) attention_tile_join_kernel(const __grid_constant__ AttnParams p) {
    using S = TileShape<D, TC>;
    constexpr int kRows = 4, kVec = D / 128;
    pdl_trigger();
    pdl_wait();
    if (blockIdx.y == 0) zero_blind_rows<T>(p);
    const int pairs = gridDim.x;
    if (tile_marks(p, pairs)[2 * blockIdx.x] | tile_marks(p, pairs)[2 * blockIdx.x + 1]) odd_rows_of_run<T, TC>(p);
    const PartHead* heads = reinterpret_cast<const PartHead*>(p.part);
    const float* parts = tile_parts(p, pairs);
    const int w0 = blockIdx.x, lane = threadIdx.x & 31, n0 = blockIdx.y * 8 * kRows + (threadIdx.x >> 5) * kRows;
    int which = -1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (heads[2 * w0 + i].begins == 1 && heads[2 * w0 + i].ends == 0) which = i;
    if (which < 0) return;
    const PartHead h = heads[2 * w0 + which];
    const int rows = min(kRows, h.tokens * p.group - n0);
    if (rows <= 0) return;
    const int count = h.last - w0 + 1;
    auto part = [&](int i) { return parts + (int64_t)(i == 0 ? 2 * w0 + which : 2 * (w0 + i)) * S::kPart; };
    float m[kRows], l[kRows] = {};
    float4 acc[kRows][kVec];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        m[r] = -INFINITY;
#pragma unroll
        for (int c = 0; c < kVec; ++c) acc[r][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = lane; i < count; i += 32)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (r < rows) m[r] = fmaxf(m[r], part(i)[n0 + r]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) m[r] = warp_max(m[r]);
    for (int i = 0; i < count; ++i) {
        const float* one = part(i);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (r >= rows) continue;
            const float weight = tile_exp2(one[n0 + r] - (m[r] == -INFINITY ? 0.f : m[r]));
            l[r] = fmaf(weight, one[kTileRows + n0 + r], l[r]);
#pragma unroll
            for (int c = 0; c < kVec; ++c) {
                if (c * 128 + lane * 4 >= p.c.head_dim) continue;
                const float4 v = *reinterpret_cast<const float4*>(one + 2 * kTileRows + (int64_t)(n0 + r) * D + c * 128 + lane * 4);
                acc[r][c].x = fmaf(weight, v.x, acc[r][c].x); acc[r][c].y = fmaf(weight, v.y, acc[r][c].y);
                acc[r][c].z = fmaf(weight, v.z, acc[r][c].z); acc[r][c].w = fmaf(weight, v.w, acc[r][c].w);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= rows) continue;
        const int n = n0 + r, tok = n / p.group, qh = h.head * p.group + n - tok * p.group;
        T* out = reinterpret_cast<T*>(p.out) + (int64_t)(h.first_row + tok) * p.os[0] + (int64_t)qh * p.os[1];
        bool odd = false;
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
            const float v[4] = {acc[r][c].x, acc[r][c].y, acc[r][c].z, acc[r][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = c * 128 + lane * 4 + e;
                if (d >= p.c.head_dim) continue;
                const float x = l[r] == 0.f ? 0.f : v[e] / l[r];
                odd |= l[r] == l[r] && !(fabsf(x) < INFINITY);
                store_elem(out + d, x);
            }
        }
        if (h.tokens > 1 && __any_sync(kFull, odd)) {
            __syncwarp();
            row_again<T, TC>(p, h.seq, h.first_row, h.pos0, h.tokens, tok, qh);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// Rows per tensor copy: the largest power of two up to 64 that divides the page size (a copy stays within a page, and copies start
// at its multiples); 0 below 8, the height of the swizzle's pattern.
static int unit_rows(int page_size) {
    int unit = 64;
    while (unit >= 8 && page_size % unit) unit >>= 1;
    return unit >= 8 ? unit : 0;
}

// Box of [unit rows][64 columns] of one head of one page; columns beyond head_dim and pages beyond the last read as zeros.
static bool page_map(const void* base, const fk_kv_cache& c, const int64_t* stride, int unit, CUtensorMap* out) {
    const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_size, (uint64_t)c.kv_heads, (uint64_t)c.pages};
    const uint64_t strides[3] = {(uint64_t)stride[2] * 2, (uint64_t)stride[1] * 2, (uint64_t)stride[0] * 2};
    const uint32_t box[4] = {64, (uint32_t)unit, 1, 1};
    return cache_tensor_map(base, c.dtype, 4, dims, strides, box, out);
}

template <int D, typename T, typename TC, bool TMA>
static int launch_tile(const AttnParams& p, const CUtensorMap& key_map, const CUtensorMap& value_map, int unit, cudaStream_t stream) {
    using S = TileShape<D, TC>;
    auto kern = attention_tile_kernel<D, T, TC, TMA>;
    static std::atomic<uint64_t> allowed;
    FK_CUDA_OK(allow_smem(kern, S::kSmem, allowed), "attention (tile) attr");
    cudaLaunchConfig_t cfg{};
    const int pairs = sm_count() / 2;
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    FK_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p, key_map, value_map, unit), "attention (tile) launch");
    FK_LAUNCH_OK("attention (tile) launch");
    FK_CUDA_OK(launch_pdl(attention_tile_join_kernel<D, T, TC>, dim3((unsigned)pairs, kTileRows / 32), dim3(256), 0, stream, p), "attention (tile) join launch");
    FK_LAUNCH_OK("attention (tile) join launch");
    return FK_OK;
}

template <int D, typename T, typename TC>
static int tile(AttnParams p, size_t* need, cudaStream_t stream) {
    p.tile_tokens = kTileRows / p.group;
    if (need) {
        const int pairs = sm_count() / 2;
        *need = tile_head_bytes(pairs) + (size_t)pairs * 2 * TileShape<D, TC>::kPart * sizeof(float);
        return FK_OK;
    }
    CUtensorMap key_map{}, value_map{};
    if constexpr (sizeof(TC) == 2) {
        // Tensor copies wherever pages and strides allow them (2048 tokens at 16384: with rows copied by threads 785 us)
        const int unit = unit_rows(p.c.page_size);
        if (unit > 0 && page_map(p.c.key, p.c, p.c.key_stride, unit, &key_map) && page_map(p.c.value, p.c, p.c.value_stride, unit, &value_map))
            return launch_tile<D, T, TC, true>(p, key_map, value_map, unit, stream);
    }
    return launch_tile<D, T, TC, false>(p, key_map, value_map, 0, stream);
}

template <typename T, typename TC>
static int tile_dim(const AttnParams& p, size_t* need, cudaStream_t stream) {
    return p.c.head_dim <= 128 ? tile<128, T, TC>(p, need, stream) : tile<256, T, TC>(p, need, stream);
}

bool attention_tile_supported(const AttnParams& p, int dtype) {
    if (dtype != FK_BF16 && dtype != FK_F16) return false;
    if (p.c.head_dim % 8 != 0 || p.group > kTileRows) return false;
    const int cb = dtype_bytes(p.c.dtype), align = cb == 1 ? 8 : 16;
    return groups_aligned(p.c.key, p.c.key_stride, 3, cb, align) && groups_aligned(p.c.value, p.c.value_stride, 3, cb, align) && groups_aligned(p.query, p.qs, 2, 2, 16);
}

// need != null: only the workspace's size
int attention_tile(const AttnParams& p, int dtype, size_t* need, cudaStream_t stream) {
    if (dtype == FK_BF16)
        return p.c.dtype == FK_E4M3 ? tile_dim<__nv_bfloat16, __nv_fp8_e4m3>(p, need, stream) : tile_dim<__nv_bfloat16, __nv_bfloat16>(p, need, stream);
    return p.c.dtype == FK_E4M3 ? tile_dim<__half, __nv_fp8_e4m3>(p, need, stream) : tile_dim<__half, __half>(p, need, stream);
}

}  // namespace fk
