// Items of paged attention (sequence, key/value head, tile of new tokens) and the tiles of keys that each of them reads, in one
// order that every block and warp derives for itself from the lengths on the device.
#pragma once

#include "attention.cuh"

namespace fk {

// Sequence s of a call: rows [first, first + n), the token of row r at position base + r.
struct SeqRows { int first, n, base; };

__device__ __forceinline__ SeqRows rows_of_seq(const AttnParams& p, int s) {
    SeqRows r;
    if (p.starts == nullptr) {
        r.first = s;
        r.n = s < p.rows ? 1 : 0;
        r.base = max(p.c.lengths[s], 0) - 1 - s;
        return r;
    }
    const int a = p.starts[s], b = p.starts[s + 1];
    r.first = min(max(a, 0), p.rows);
    const int end = min(max(b, 0), p.rows);
    r.n = max(0, end - r.first);
    r.base = max(p.c.lengths[s], 0) - end;          // no position exceeds lengths - 1, whatever the starts hold
    return r;
}

// Key tiles of KT positions that some token at pos0 .. pos1 sees: tiles 0 .. sink_tiles-1, then lo_tile .. ; count in all.
struct TileSpan { int sink_tiles, lo_tile, count, end; };

template <int KT>
__device__ __forceinline__ TileSpan span_of(const AttnParams& p, int pos0, int pos1) {
    TileSpan s{0, 0, 0, 0};
    s.end = min(pos1 + 1, p.c.max_pages * p.c.page_size);
    if (s.end <= 0) return s;
    const int lo = min(window_start(p, pos0), s.end);
    const int hi_tile = (s.end + KT - 1) / KT;
    const int sink_tiles = (min(p.sinks, lo) + KT - 1) / KT, lo_tile = lo / KT;
    if (sink_tiles >= lo_tile) {
        s.count = hi_tile;
    } else {
        s.sink_tiles = sink_tiles;
        s.lo_tile = lo_tile;
        s.count = sink_tiles + (lo < s.end ? hi_tile - lo_tile : 0);
    }
    return s;
}

__device__ __forceinline__ bool sees(const AttnParams& p, int pos, int j) {
    return j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
}

// Bits of 32 consecutive positions from j0 on that a token at position pos sees.
__device__ __forceinline__ uint32_t seen_bits(const AttnParams& p, int pos, int j0) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };       // positions j0 .. j0 + n - 1
    const uint32_t past = below(pos - j0 + 1);
    if (p.window == 0) return past;
    return past & (~below(pos - p.window - j0 + 1) | below(p.sinks - j0));
}

// A position in the order (sequence, head, tile of tokens, key tile).  All lanes of a warp hold the same.
template <int KT>
struct ItemCursor {
    int seq, head, tile;       // item: tokens [tile * p.tile_tokens, ..) of the sequence
    SeqRows rows;
    int pos0, pos1;            // first and last token's position
    TileSpan span;
    int k;                     // key tile of the item

    __device__ __forceinline__ int tokens(const AttnParams& p) const { return min(p.tile_tokens, rows.n - tile * p.tile_tokens); }
    __device__ __forceinline__ int first_row(const AttnParams& p) const { return rows.first + tile * p.tile_tokens; }
    __device__ __forceinline__ int key0() const { return (k < span.sink_tiles ? k : span.lo_tile + k - span.sink_tiles) * KT; }
    __device__ __forceinline__ bool some_row_sees(const AttnParams& p, int j) const {
        return j < span.end && (p.window == 0 || j >= window_start(p, pos0) || j < p.sinks);
    }
    __device__ __forceinline__ void set_item(const AttnParams& p) {
        pos0 = rows.base + first_row(p);
        pos1 = pos0 + tokens(p) - 1;
        span = span_of<KT>(p, pos0, pos1);
    }
    // to the first key tile of the next item that has any
    __device__ __forceinline__ void next_item(const AttnParams& p) {
        k = 0;
        while (true) {
            if (++tile * p.tile_tokens >= rows.n) {
                tile = 0;
                if (rows.n == 0 || ++head >= p.c.kv_heads) {
                    head = 0;
                    do {
                        if (++seq >= p.c.seqs) return;
                        rows = rows_of_seq(p, seq);
                    } while (rows.n == 0);
                }
            }
            set_item(p);
            if (span.count > 0) return;
        }
    }
};

// Key tiles of one head's items of a sequence.
template <int KT>
__device__ __forceinline__ int64_t seq_tiles(const AttnParams& p, const SeqRows& r) {
    int64_t sum = 0;
    for (int t = 0; t < r.n; t += p.tile_tokens) {
        const int pos0 = r.base + r.first + t;
        sum += span_of<KT>(p, pos0, pos0 + min(p.tile_tokens, r.n - t) - 1).count;
    }
    return sum;
}

// The order's extent and, in shared memory, where each sequence ends in it: upto[s] key tiles up to and with sequence s, for as many
// sequences as `room` holds (others are counted again by locate).  Every thread of the block calls it; `scratch` holds two words
// per warp.
template <int KT>
__device__ __forceinline__ int64_t plan_tiles(const AttnParams& p, int64_t* scratch, int64_t* upto, int room) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int64_t all = 0;
    for (int s0 = 0, turn = 0; s0 < p.c.seqs; s0 += blockDim.x, turn ^= 1) {
        const int s = s0 + threadIdx.x;
        int64_t mine = 0;
        if (s < p.c.seqs) {
            const SeqRows r = rows_of_seq(p, s);
            if (r.n > 0) mine = seq_tiles<KT>(p, r) * p.c.kv_heads;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(kFull, mine, o);
            if (lane >= o) mine += up;
        }
        if (lane == 31) scratch[turn * warps + warp] = mine;
        __syncthreads();
        int64_t before = all;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) before += scratch[turn * warps + w];
            all += scratch[turn * warps + w];
        }
        if (s < p.c.seqs && s < room) upto[s] = before + mine;
    }
    __syncthreads();
    return all;
}

// Cursor at key tile `target` of the order (target < the extent); a whole warp calls it.
template <int KT>
__device__ __forceinline__ void locate(const AttnParams& p, int64_t target, const int64_t* upto, int room, ItemCursor<KT>& c) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int s0 = 0; s0 < p.c.seqs; s0 += 32) {
        const int s = s0 + lane;
        int64_t end = 0;                         // of this lane's sequence
        if (s0 + 32 <= room || p.c.seqs <= room) {
            if (s < p.c.seqs) end = upto[s];
        } else {
            if (s < p.c.seqs) {
                const SeqRows r = rows_of_seq(p, s);
                if (r.n > 0) end = seq_tiles<KT>(p, r) * p.c.kv_heads;
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(kFull, end, o);
                if (lane >= o) end += up;
            }
            end += before;
        }
        const unsigned past = __ballot_sync(kFull, s < p.c.seqs && end > target);
        if (past == 0) {
            before = __shfl_sync(kFull, end, min(31, p.c.seqs - s0 - 1));
            continue;
        }
        const int at = __ffs(past) - 1;
        const int64_t start = at > 0 ? __shfl_sync(kFull, end, at > 0 ? at - 1 : 0) : before;
        int64_t rest = target - start;
        const int64_t per_head = (__shfl_sync(kFull, end, at) - start) / p.c.kv_heads;
        c.seq = s0 + at;
        c.rows = rows_of_seq(p, c.seq);
        c.head = (int)(rest / per_head);
        rest -= c.head * per_head;
        for (c.tile = 0;; ++c.tile) {
            c.set_item(p);
            if (rest < c.span.count) break;
            rest -= c.span.count;
        }
        c.k = (int)rest;
        return;
    }
}

// Zeros for the rows that see nothing, and for those behind the last sequence if asked for.  Sequences are dealt to the blocks.
template <typename T>
__device__ __forceinline__ void zero_blind_rows(const AttnParams& p) {
    const int width = p.q_heads * p.c.head_dim;
    T* out = reinterpret_cast<T*>(p.out);
    auto clear = [&](int row) {
        for (int i = threadIdx.x; i < width; i += blockDim.x) {
            const int a = i / p.c.head_dim;
            store_elem(out + row * p.os[0] + a * p.os[1] + (i - a * p.c.head_dim), 0.f);
        }
    };
    for (int s = blockIdx.x; s < p.c.seqs; s += gridDim.x) {
        const SeqRows r = rows_of_seq(p, s);
        if (r.n == 0) continue;
        const int pos = r.base + r.first;
        // only a sequence shorter than its rows, or one that reaches beyond its table, has such rows
        if (pos >= 0 && (int64_t)pos + r.n <= p.c.max_pages * p.c.page_size) continue;
        for (int i = 0; i < r.n; ++i)
            if (span_of<1>(p, pos + i, pos + i).count == 0) clear(r.first + i);
    }
    if (p.zero_rest) {
        const int used = p.starts ? min(max(p.starts[p.c.seqs], 0), p.rows) : min(p.c.seqs, p.rows);
        const int unused = p.starts ? min(max(p.starts[0], 0), p.rows) : 0;         // 0 unless the starts are no starts
        for (int row = blockIdx.x; row < p.rows; row += gridDim.x)
            if (row < unused || row >= used) clear(row);
    }
}

// Columns of the values at positions [from, to) of a sequence that are not finite (NAN_ONLY: not a number), one bit per group of 32 columns,
// for this lane's column of each.  A whole warp: a lane looks a position up, then the rows are read one after the other.
template <typename TC, bool NAN_ONLY>
__device__ __forceinline__ unsigned odd_columns(const AttnParams& p, int seq, int head, int from, int to) {
    const int lane = threadIdx.x & 31, D = p.c.head_dim;
    const TC* values = reinterpret_cast<const TC*>(p.c.value);
    unsigned odd = 0;
    for (int64_t j0 = max(from, 0); j0 < to; j0 += 32) {
        int in_page = 0, page = -1;
        if (j0 + lane < to) page = page_of(p.c, seq, (int)(j0 + lane), in_page);
        const int64_t off = page < 0 ? -1 : row_offset(p.c.value_stride, page, head, in_page);
        float scale = 1.f;
        if (sizeof(TC) == 1 && page >= 0) scale = p.c.value_scale[row_offset(p.c.value_scale_stride, page, head, in_page)];
#pragma unroll 4
        for (int i = 0; i < 32; ++i) {
            const int64_t row = __shfl_sync(kFull, off, i);
            const float one = __shfl_sync(kFull, scale, i);
            if (row < 0) continue;
#pragma unroll
            for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
                if (c * 32 + lane < D) {
                    const float v = load_elem(values + row + c * 32 + lane) * one;
                    if (NAN_ONLY ? v != v : !(fabsf(v) < INFINITY)) odd |= 1u << c;
                }
        }
    }
    return odd;
}

// A row of an item of several tokens, once more by itself and exactly if its result owes a number that is not finite to a key that it does
// not see: such a key's value may have entered the row's product as 0 * infinity.  Only keys that some tokens of the item see and others
// do not can: those of the item's own tokens, and those that the window leaves behind.  They are looked at first, so that numbers that
// are not finite and that the row does see cost no second pass over its keys; nor do columns in which it sees a NaN among them anyway.  A whole warp;
// the item's tokens are at positions pos0 .. pos0 + tokens - 1, the row is the tok-th of them.
template <typename T, typename TC>
__device__ __noinline__ void row_again(const AttnParams& p, int seq, int first_row, int pos0, int tokens, int tok, int qh) {
    const int lane = threadIdx.x & 31, D = p.c.head_dim, row = first_row + tok, pos = pos0 + tok, pos1 = pos0 + tokens - 1, head = qh / p.group;
    T* out = reinterpret_cast<T*>(p.out) + row * p.os[0] + qh * p.os[1];
    bool odd = false;
#pragma unroll
    for (int c = 0; c < FK_MAX_HEAD_DIM / 32; ++c)
        if (c * 32 + lane < D) odd |= !(fabsf(to_float(out[c * 32 + lane])) < INFINITY);
    if (!__any_sync(kFull, odd)) return;
    const int all = p.c.max_pages * p.c.page_size, lo = window_start(p, pos);
    unsigned hidden = odd_columns<TC, false>(p, seq, head, pos + 1, min(pos1 + 1, all));
    if (p.window > 0) hidden |= odd_columns<TC, false>(p, seq, head, max(window_start(p, pos0), p.sinks), min(lo, all));
    if (!__any_sync(kFull, hidden != 0)) return;
    hidden &= ~odd_columns<TC, true>(p, seq, head, max(pos0, lo), min(pos + 1, all));
    if (p.window > 0) hidden &= ~odd_columns<TC, true>(p, seq, head, lo, min(min(window_start(p, pos1), pos + 1), all));
    if (!__any_sync(kFull, hidden != 0)) return;
    const T* query = reinterpret_cast<const T*>(p.query) + row * p.qs[0] + qh * p.qs[1];
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = 8 * lane + e < D ? load_elem(query + 8 * lane + e) * p.scale_log2 : 0.f;
    RowSums r;
    warp_row<TC>(p, q, seq, head, pos, r);       // the kernels of tiles only take calls whose rows allow its wide loads
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (8 * lane + e < D) store_elem(out + 8 * lane + e, r.l == 0.f ? 0.f : r.acc[e] / r.l);
}

// Runs of key tiles: worker w of `workers` has [w * all / workers, (w + 1) * all / workers), or `least` tiles if that is more.
struct Runs {
    int64_t all, workers;
    int least;
    __device__ __forceinline__ bool even() const { return all >= workers * least; }
    __device__ __forceinline__ int64_t begin(int64_t w) const { return even() ? w * all / workers : min(w * least, all); }
    __device__ __forceinline__ int worker_of(int64_t tile) const { return (int)(even() ? ((tile + 1) * workers - 1) / all : tile / least); }
};

// What a worker's partial result belongs to.
struct PartHead {
    int first_row, tokens, head, seq, pos0;
    int begins, ends;                           // the run has the item's first / last key tile
    int last;                                   // worker whose run has the item's last key tile
};

}  // namespace fk
