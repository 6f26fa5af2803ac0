// How the attention over a paged cache is dealt out to CTAs. A unit is a sequence, a key head and a tile of rows, where a row is a query
// head of the group that shares the key head, at a token of the pass (row = token * group + head): they read the same keys. Its
// work is counted in blocks of keys, and unit_cost of them for what a unit costs whatever its length (queries, the first reads, its end). All
// units' work, one behind the other, is cut into equal shares, so that long and short sequences, prompts and single tokens, few and many of
// them all fill the device; a unit that a cut goes through is put together from its parts by a second launch. (Without unit_cost one CTA had
// the eight units of a sequence of 50 keys among 37 of up to 6000, and the others waited for it: 36 us
// where it takes 25.) Lengths are known on the device alone, so every CTA forms the sums by itself.
#pragma once
#include "ptx.cuh"
#include "round_ops.h"

namespace mk {

// Quotients of any x below 2^31 by the page size and the group: inverses are 2^(31 + b) / n, rounded up, 2^b being at least n.
__device__ __forceinline__ uint32_t kv_page_of(const KvAttendArgs& a, uint32_t x) { return (uint32_t)(((uint64_t)x * a.page_inverse) >> a.page_shift); }
__device__ __forceinline__ uint32_t kv_token_of(const KvAttendArgs& a, uint32_t row) { return (uint32_t)(((uint64_t)row * a.group_inverse) >> a.group_shift); }

struct KvSeq {
    uint32_t first, n; // rows of the pass that are this sequence's tokens
    uint32_t len;      // tokens, the last n of which are the rows'
    uint32_t keys;     // of them that the block table has columns for
};

__device__ __forceinline__ KvSeq kv_seq(const KvAttendArgs& a, uint32_t s)
{
    const int64_t most = a.n_tokens, held = (int64_t)a.table_cols * a.c.page_size;
    int64_t from = __ldg(a.query_start + s), to = __ldg(a.query_start + s + 1), len = __ldg(a.kv_len + s);
    from = from < 0 ? 0 : from > most ? most : from;
    to = to < from ? from : to > most ? most : to;
    len = len < 0 ? 0 : len;
    return KvSeq{(uint32_t)from, (uint32_t)(to - from), (uint32_t)len, (uint32_t)(len > held ? held : len)};
}

// The blocks of `each` keys that a tile of rows has to look at: [from, to), at least one, so that a tile that sees nothing is a unit too.
struct KvBlocks {
    uint32_t from, to;
};

__device__ __forceinline__ KvBlocks kv_blocks(const KvAttendArgs& a, const KvSeq& q, uint32_t row0, uint32_t rows, uint32_t each)
{
    const int32_t back = (int32_t)q.len - (int32_t)q.n;                     // the position of the pass's first token
    const int32_t end = min(back + (int32_t)(kv_token_of(a, row0 + rows - 1u)) + 1, (int32_t)q.keys);
    const int32_t first = back + (int32_t)kv_token_of(a, row0) + 1;
    const uint32_t lo = a.window && first > (int32_t)a.window ? (uint32_t)first - a.window : 0u;
    const uint32_t from = lo / each, to = end < 0 ? 0u : ((uint32_t)end + each - 1u) / each;
    return KvBlocks{from, to > from ? to : from + 1u};
}

// A sequence's rows, or 0 where it is not this launch's.
__device__ __forceinline__ uint32_t kv_rows(const KvAttendArgs& a, const KvSeq& q)
{
    const uint32_t rows = q.n * a.group;
    return rows < a.rows_from || rows > a.rows_to ? 0u : rows;
}

// A unit's work.
__device__ __forceinline__ uint32_t kv_tile_blocks(const KvAttendArgs& a, const KvSeq& q, uint32_t rows, uint32_t row0, uint32_t tile, uint32_t each)
{
    if (row0 >= rows)
        return 0;
    const KvBlocks b = kv_blocks(a, q, row0, min(tile, rows - row0), each);
    return b.to - b.from + a.unit_cost;
}

// Of each lane's sequence: the work of one key head, all of its tiles of rows together. A sequence of many tiles (a prompt) is counted by the
// warp. By whole warps.
__device__ __forceinline__ uint64_t kv_seq_blocks(const KvAttendArgs& a, const KvSeq& q, uint32_t rows, uint32_t tile, uint32_t each)
{
    constexpr uint32_t few = 4; // tiles that a lane counts by itself
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t sum = 0;
    for (uint32_t i = 0; i < few; ++i)
        sum += kv_tile_blocks(a, q, rows, i * tile, tile, each);
    uint32_t many = __ballot_sync(~0u, rows > few * tile);
    while (many) {
        const int i = __ffs(many) - 1;
        many &= many - 1u;
        const KvSeq other{0u, __shfl_sync(~0u, q.n, i), __shfl_sync(~0u, q.len, i), __shfl_sync(~0u, q.keys, i)};
        const uint32_t its = __shfl_sync(~0u, rows, i);
        uint64_t x = 0;
        for (uint32_t r = lane * tile; r < its; r += 32u * tile)
            x += kv_tile_blocks(a, other, its, r, tile, each);
        __syncwarp();
        x = ((uint64_t)__reduce_add_sync(~0u, (uint32_t)(x >> 26)) << 26) + __reduce_add_sync(~0u, (uint32_t)x & 0x3ffffffu); // (x below 2^53)
        sum = lane == (uint32_t)i ? x : sum;
    }
    return sum;
}

// Where share i of n of a whole begins: shares differ by one at most.
__device__ __forceinline__ uint64_t kv_cut(uint64_t total, uint32_t n, uint32_t i)
{
    if (total >> 32) // (a division in 64 bits takes some hundred instructions)
        return total / n * i + min((uint64_t)i, total % n);
    const uint32_t each = (uint32_t)total / n, more = (uint32_t)total - each * n;
    return (uint64_t)each * i + min(i, more);
}

// What a row's weights p_j v_j (v_j: the scale of key j's values) are held in, as fp16: a weight of 1 is 2^unit, where exponents of p are those
// of its scores. Whatever the row does not see, and whatever scales there are elsewhere, has no part in it: its largest weight so far is from 2^7 to
// 2^15, so that one is rounded by 2^-11 of it down to 2^-21 of the largest. `high`: log2 of the largest weight of a block (-inf: none), too large by
// kHighSlack at most; `ref`: that of p = 1, which a unit is at most 2^126 below, so that what it is multiplied by is a number. +inf: no weight yet.
constexpr float kHighSlack = 3.0f;
__device__ __forceinline__ float kv_unit(float unit, float high, float ref)
{
    if (high > unit + 15.0f || (unit == INFINITY && high > -INFINITY))
        unit = high - (7.0f + kHighSlack);
    return fmaxf(unit, ref - 126.0f);
}
// What outputs in one unit are worth in another.
__device__ __forceinline__ float kv_worth(float unit, float in) { return unit == INFINITY ? 0.0f : ex2_approx(unit - in); }

// A CTA's share of all work, [at, end), and the unit that it begins in, `skip` behind the unit's begin. kv_take gives one segment after the
// other. A unit's blocks come first, what else it costs behind them.
struct KvWalk {
    uint64_t at, end, total;
    uint32_t ctas; // that have a share
    uint32_t sq, head, row0, skip;
};

// By all Threads of a CTA; scratch: 40 words of 8 bytes.
template <uint32_t Threads>
__device__ KvWalk kv_find(const KvAttendArgs& a, uint32_t tile, uint32_t each, uint32_t ctas_most, uint64_t* scratch, uint32_t cta)
{
    const uint32_t tid = threadIdx.x, lane = tid & 31u, mine = (a.n_seq + Threads - 1) / Threads;
    auto of = [&](uint32_t k) -> uint64_t { // blocks of this thread's sequence k, all heads
        const uint32_t s = tid * mine + k;
        const KvSeq q = s < a.n_seq ? kv_seq(a, s) : KvSeq{0, 0, 0, 0};
        return kv_seq_blocks(a, q, s < a.n_seq ? kv_rows(a, q) : 0u, tile, each) * a.c.n_heads;
    };
    uint64_t sum = 0;
    for (uint32_t k = 0; k < mine; ++k)
        sum += of(k);
    uint64_t run = sum;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, run, d);
        if (lane >= d)
            run += y;
    }
    if (lane == 31u)
        scratch[tid / 32u] = run;
    __syncthreads();
    KvWalk w;
    uint64_t front = 0;
    w.total = 0;
    for (uint32_t i = 0; i < Threads / 32u; ++i) {
        front += i < tid / 32u ? scratch[i] : 0ull;
        w.total += scratch[i];
    }
    w.ctas = ctas_most;
    if (w.total < (uint64_t)a.blocks_least * ctas_most)
        w.ctas = ((uint32_t)w.total + a.blocks_least - 1u) / a.blocks_least;
    const bool has = cta < w.ctas;
    w.at = has ? kv_cut(w.total, w.ctas, cta) : 0;
    w.end = has ? kv_cut(w.total, w.ctas, cta + 1u) : 0;
    uint64_t at = front + run - sum; // of this thread's first sequence
    if (__any_sync(~0u, has && w.at >= at && w.at < at + sum)) {
        for (uint32_t k = 0; k < mine; ++k) {
            const uint64_t n = mine == 1u ? sum : of(k);
            if (has && w.at >= at && w.at < at + n) {
                scratch[32] = tid * mine + k;
                scratch[33] = w.at - at;
                scratch[34] = n;
            }
            at += n;
        }
    }
    __syncthreads();
    if (has && tid < 32u) { // the head and, 32 at a time, the tile
        const uint32_t s = (uint32_t)scratch[32];
        const uint64_t off = scratch[33], all = scratch[34];
        const KvSeq q = kv_seq(a, s);
        const uint32_t rows = kv_rows(a, q);
        const uint64_t per_head = all >> 32 ? all / a.c.n_heads : (uint32_t)all / a.c.n_heads;
        const uint32_t head = all >> 32 ? (uint32_t)(off / per_head) : (uint32_t)off / (uint32_t)per_head;
        uint64_t left = off - head * per_head;
        for (uint32_t r0 = 0; r0 < rows; r0 += 32u * tile) {
            const uint32_t r = r0 + lane * tile, n = kv_tile_blocks(a, q, rows, r, tile, each);
            uint32_t upto = n;
#pragma unroll
            for (uint32_t d = 1; d < 32; d <<= 1) {
                const uint32_t y = __shfl_up_sync(~0u, upto, d);
                upto += lane >= d ? y : 0u;
            }
            if (left < upto && left >= upto - n) {
                scratch[35] = head;
                scratch[36] = r;
                scratch[37] = left - (upto - n); // (32 tiles' work is below 2^32)
            }
            const uint32_t these = __shfl_sync(~0u, upto, 31);
            if (left < these)
                break;
            left -= these;
        }
    }
    __syncthreads();
    w.sq = (uint32_t)scratch[32];
    w.head = (uint32_t)scratch[35];
    w.row0 = (uint32_t)scratch[36];
    w.skip = (uint32_t)scratch[37];
    return w;
}

// A unit, and the blocks [from, to) of it that a CTA has.
struct KvSegment {
    KvSeq seq;
    KvBlocks blocks; // all of the unit's
    uint32_t sq, head, row0, rows, from, to;
    __device__ __forceinline__ bool whole() const { return from == blocks.from && to == blocks.to; }
    // Where a part of a unit goes. A CTA has two places: for a unit that another one began, and for one that it begins.
    __device__ __forceinline__ uint32_t place(uint32_t cta) const { return 2u * cta + (from == blocks.from); }
};

// The walk's next segment; false behind the last. `g` is the one before.
__device__ __forceinline__ bool kv_take(const KvAttendArgs& a, KvWalk& w, KvSegment& g, bool first, uint32_t tile, uint32_t each)
{
    while (w.at < w.end) {
        if (first || w.row0 == 0) { // (a sequence begins, or a head)
            g.seq = kv_seq(a, w.sq);
            while (kv_rows(a, g.seq) == 0) {
                if (++w.sq >= a.n_seq) // (not while lengths stay as they were)
                    return false;
                g.seq = kv_seq(a, w.sq);
            }
            first = false;
        }
        const uint32_t rows = g.seq.n * a.group;
        g.sq = w.sq;
        g.head = w.head;
        g.row0 = w.row0;
        g.rows = min(tile, rows - w.row0);
        g.blocks = kv_blocks(a, g.seq, g.row0, g.rows, each);
        const uint32_t n = g.blocks.to - g.blocks.from, all = n + a.unit_cost;
        const uint32_t upto = w.end - w.at < all - w.skip ? w.skip + (uint32_t)(w.end - w.at) : all;
        g.from = g.blocks.from + min(w.skip, n);
        g.to = g.blocks.from + min(upto, n);
        w.at += upto - w.skip;
        w.skip = 0;
        w.row0 += tile;
        if (w.row0 >= rows) {
            w.row0 = 0;
            if (++w.head == a.c.n_heads) {
                w.head = 0;
                ++w.sq;
            }
        }
        if (g.from < g.to)
            return true;
    }
    return false;
}

} // namespace mk
