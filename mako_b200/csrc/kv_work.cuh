// How the attention over a paged cache is dealt out to CTAs. A unit is a sequence, a key head and a tile of rows, where a row is a query
// head of the group that shares the key head, at a token of the pass (row = token * group + head): they read the same keys. Its
// work is counted in blocks of keys. All units' blocks, one behind the other, are cut into equal shares, so that long and short
// sequences, prompts and single tokens, few and many of them all fill the device; a unit that a cut goes through is put together from
// its parts by a second launch. Lengths are known on the device alone, so every CTA forms the sums by itself.
#pragma once
#include "round_ops.h"

namespace mk {

struct KvSeq {
    uint32_t first, n; // rows of the pass that are this sequence's tokens
    uint32_t len;      // keys
};

__device__ __forceinline__ KvSeq kv_seq(const KvAttendArgs& a, uint32_t s)
{
    const int64_t most = a.n_tokens, held = (int64_t)a.table_cols * a.c.page_size;
    int64_t from = __ldg(a.query_start + s), to = __ldg(a.query_start + s + 1), len = __ldg(a.kv_len + s);
    from = from < 0 ? 0 : from > most ? most : from;
    to = to < from ? from : to > most ? most : to;
    len = len < 0 ? 0 : len > held ? held : len;
    return KvSeq{(uint32_t)from, (uint32_t)(to - from), (uint32_t)len};
}

// The blocks of `each` keys that a tile of rows has to look at: [from, to), at least one, so that a tile that sees nothing is a unit too.
struct KvBlocks {
    uint32_t from, to;
};

__device__ __forceinline__ KvBlocks kv_blocks(const KvAttendArgs& a, const KvSeq& q, uint32_t row0, uint32_t rows, uint32_t each)
{
    const int64_t back = (int64_t)q.len - q.n; // the position of the pass's first token
    const int64_t end = back + (row0 + rows - 1u) / a.group + 1;
    const uint32_t hi = end < 0 ? 0u : end > q.len ? q.len : (uint32_t)end;
    const int64_t begin = a.window ? back + row0 / a.group - (int64_t)a.window + 1 : 0;
    const uint32_t lo = begin < 0 ? 0u : (uint32_t)begin, from = lo / each, to = (hi + each - 1u) / each;
    return KvBlocks{from, to > from ? to : from + 1u};
}

// Of a sequence: blocks of one key head, all of its tiles of rows together. 0 for a sequence that is not this launch's.
__device__ __forceinline__ uint32_t kv_seq_blocks(const KvAttendArgs& a, const KvSeq& q, uint32_t tile, uint32_t each)
{
    const uint32_t rows = q.n * a.group;
    if (rows < a.rows_from || rows > a.rows_to)
        return 0;
    uint32_t sum = 0;
    for (uint32_t r = 0; r < rows; r += tile) {
        const KvBlocks b = kv_blocks(a, q, r, min(tile, rows - r), each);
        sum += b.to - b.from;
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

struct KvAt {
    uint32_t seq;
    uint64_t off;   // blocks into the sequence
};

// Where the block `at` of all lies, and how many there are, by all Threads of a CTA; scratch: Threads + 8 words of 8 bytes.
template <uint32_t Threads>
__device__ KvAt kv_find(const KvAttendArgs& a, uint32_t tile, uint32_t each, uint32_t ctas_most, uint32_t blocks_least, uint64_t* scratch,
                        uint32_t cta, uint64_t& begin, uint64_t& end, uint64_t& total, uint32_t& ctas)
{
    const uint32_t tid = threadIdx.x, lane = tid & 31u, mine = (a.n_seq + Threads - 1) / Threads;
    const uint32_t s0 = min(tid * mine, a.n_seq), s1 = min(s0 + mine, a.n_seq);
    uint64_t sum = 0;
    for (uint32_t s = s0; s < s1; ++s)
        sum += (uint64_t)kv_seq_blocks(a, kv_seq(a, s), tile, each) * a.c.n_heads;
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
    uint64_t front = 0;
    total = 0;
    for (uint32_t w = 0; w < Threads / 32u; ++w) {
        if (w < tid / 32u)
            front += scratch[w];
        total += scratch[w];
    }
    ctas = ctas_most;
    if (total < (uint64_t)blocks_least * ctas_most)
        ctas = ((uint32_t)total + blocks_least - 1u) / blocks_least;
    begin = ctas ? kv_cut(total, ctas, cta) : 0;
    end = ctas ? kv_cut(total, ctas, cta + 1u) : 0;
    uint64_t at = front + run - sum; // of this thread's first sequence
    if (cta < ctas && begin >= at && begin < at + sum)
        for (uint32_t s = s0; s < s1; ++s) {
            const uint64_t has = (uint64_t)kv_seq_blocks(a, kv_seq(a, s), tile, each) * a.c.n_heads;
            if (begin < at + has) {
                scratch[32] = s;
                scratch[33] = begin - at;
                break;
            }
            at += has;
        }
    __syncthreads();
    const KvAt found{(uint32_t)scratch[32], scratch[33]};
    __syncthreads();
    return found;
}

// A unit and what of it begins at `off` of a sequence.
struct KvUnit {
    uint32_t head, row0, rows;
    KvBlocks blocks;      // all of its blocks
    uint32_t skip;        // that come before `off`
};

__device__ __forceinline__ KvUnit kv_unit(const KvAttendArgs& a, const KvSeq& q, uint32_t seq_blocks, uint64_t off, uint32_t tile, uint32_t each)
{
    KvUnit u;
    u.head = off >> 32 ? (uint32_t)(off / seq_blocks) : (uint32_t)off / seq_blocks;
    u.skip = (uint32_t)(off - (uint64_t)u.head * seq_blocks);
    const uint32_t rows = q.n * a.group;
    for (u.row0 = 0;; u.row0 += tile) {
        u.rows = min(tile, rows - u.row0);
        u.blocks = kv_blocks(a, q, u.row0, u.rows, each);
        const uint32_t has = u.blocks.to - u.blocks.from;
        if (u.skip < has)
            return u;
        u.skip -= has;
    }
}

// Quotients by the page size: x / page for any x below 2^31 (inverse: 2^(31 + shift) / page, rounded up, shift: ceil(log2(page))).
__device__ __forceinline__ uint32_t kv_page_of(const KvAttendArgs& a, uint32_t x) { return (uint32_t)(((uint64_t)x * a.page_inverse) >> a.page_shift); }

} // namespace mk
