// Log-probabilities of given tokens, the entropy and the likeliest alternatives of whole distributions (mk_token_logprobs in
// include/mako_b200.h): every logit is read once.
//
// With c = log2(e) / temperature and any shift s a row's weights are w_i = 2^(c x_i - s); log2 of a probability is c x_t - s -
// log2(sum w), and the entropy in bits log2(sum w) - sum(w (c x - s)) / sum w. Each thread keeps (s, sum w, sum w (c x - s)) of its columns,
// s being c times the largest x so far, rounded: a shift that is a little off is as good as another as long as it is the same one
// everywhere, so that what the rounding of a large c x takes away does not reach the results.
//
// Alternatives: an x on or above `line` goes into a list of (x, id) in shared memory. The line is a lower bound of the k-th largest x that the
// CTA has seen: of groups of threads' largest in the first tile, then of the list's entries after 1, 2, 4, 8, ... tiles, so that a row in
// no particular order has about k log2(tiles) entries. A row whose list runs over (an ascending one) is read again, in pieces of
// which each fits.
//
// A CTA per row; where rows are few a cluster of up to 16 of them, whose parts are put into the first one's shared memory. Instructions bound it
// beside HBM: 2048 rows of 151552 bf16 logits take 134 us (4.6 TB/s, 0.70 of the rate of a copy; 118 if nothing were ever put into a list),
// a row of 129280 fp32 logits 10.4 from a graph, 137 masked rows of 50257 fp16 27. 16-bit logits are compared two at a time before they become
// floats; weights and sums are formed two at a time. (Five CTAs an SM, 48 registers: with four 143 us, with six 137.)
#include "ptx.cuh"
#include "round_ops.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cg = cooperative_groups;

namespace mk {
namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kTileVecs = 4;            // 16-byte blocks of a thread in a tile
constexpr uint32_t kListCap = 2048 + kLogprobMaxTop; // a piece of one block a thread (8 16-bit logits), and the best before it
constexpr uint32_t kRankMax = kThreads;      // entries that are ranked against one another by a CTA
constexpr uint32_t kWarpKeys = 128;          // and by a warp
constexpr uint32_t kMaxCluster = 16;
constexpr float kLeast = -200.0f;            // exponents are held above this: 2^-200 is nothing, and nothing times it is not NaN

using Key = unsigned long long;              // larger x first, then the lower id

__device__ __forceinline__ Key make_key(float x, uint32_t id) { return ((Key)order_key(x) << 32) | (uint32_t)~id; }
__device__ __forceinline__ float key_x(Key k) { return key_to_float((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_id(Key k) { return ~(uint32_t)k; }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename F>
struct Sums {
    F shift;
    float w, wd; // sum of weights, sum of weights times exponents
};

template <typename F>
__device__ __forceinline__ Sums<F> join(const Sums<F>& a, const Sums<F>& b)
{
    const F shift = a.shift > b.shift ? a.shift : b.shift;
    const float da = fmaxf((float)(a.shift - shift), kLeast), db = fmaxf((float)(b.shift - shift), kLeast);
    const float fa = ex2_approx(da), fb = ex2_approx(db);
    return Sums<F>{shift, a.w * fa + b.w * fb, fa * (a.wd + da * a.w) + fb * (b.wd + db * b.w)};
}

struct Shared {
    Key list[kListCap];
    Key best[kLogprobMaxTop]; // in order; in the first CTA of a cluster everybody's
    Sums<float> warp[kWarps];
    uint4 handed[kWarps][kTileVecs];
    float warp_most[kWarps];
    alignas(16) float largest[kThreads];
    Key ranked[kRankMax];
    Key of_slices[kLogprobMaxTop * kMaxCluster]; // in the first CTA of a cluster: the best of each
    Sums<double> slice_sums[kMaxCluster];        // (in 64 bits: c times a mask of the type's lowest value passes fp32)
    float slice_most[kMaxCluster];
    uint32_t slice_has[kMaxCluster]; // how many, and 0x100 where the mask allows a token
    uint32_t n;        // entries that were to go into the list
    uint32_t allowed;  // not 0: the mask allows a token
    uint32_t line, line_next; // in the order of floats
};

// Logits in words of 32 bits: one fp32 number, or two of 16 bits.
template <typename T>
struct Words;
template <>
struct Words<float> {
    static constexpr uint32_t each = 1, none = 0xff800000u; // -inf
    static constexpr float least = -999424.0f;              // what smaller ones are taken for (see add)
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float2 pair(const uint32_t* w) { return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])); }
    static __device__ __forceinline__ float largest(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float value(uint32_t w, uint32_t) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t without(uint32_t w, uint32_t there) { return there & 1u ? w : none; }
    static __device__ __forceinline__ uint32_t of_least() { return __float_as_uint(least); }
};
template <>
struct Words<__nv_bfloat16> {
    static constexpr uint32_t each = 2, none = 0xff80ff80u;
    static constexpr float least = -999424.0f;   // (eight bits)
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) // (NaN loses)
    {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float2 pair(const uint32_t* w) { return make_float2(__uint_as_float(*w << 16), __uint_as_float(*w & 0xffff0000u)); }
    static __device__ __forceinline__ float largest(uint32_t a)
    {
        const float2 x = pair(&a);
        return fmaxf(x.x, x.y);
    }
    static __device__ __forceinline__ float value(uint32_t w, uint32_t i) { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }
    static __device__ __forceinline__ uint32_t without(uint32_t w, uint32_t there)
    {
        return ((there & 1u ? w : none) & 0xffffu) | ((there & 2u ? w : none) & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t of_least() { return (__float_as_uint(least) >> 16) * 0x10001u; }
};
template <>
struct Words<__half> {
    static constexpr uint32_t each = 2, none = 0xfc00fc00u;
    static constexpr float least = -65504.0f;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float2 pair(const uint32_t* w) { return __half22float2(*reinterpret_cast<const __half2*>(w)); }
    static __device__ __forceinline__ float largest(uint32_t a)
    {
        const float2 x = pair(&a);
        return fmaxf(x.x, x.y);
    }
    static __device__ __forceinline__ float value(uint32_t w, uint32_t i)
    {
        const float2 x = pair(&w);
        return i ? x.y : x.x;
    }
    static __device__ __forceinline__ uint32_t without(uint32_t w, uint32_t there)
    {
        return ((there & 1u ? w : none) & 0xffffu) | ((there & 2u ? w : none) & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t of_least() { return 0xfbfffbffu; }
};

// A CTA's columns of a row: blocks [from, to) of those that begin at the last 16-byte boundary in front of the row.
struct Columns {
    const uint4* base;
    uint32_t before;   // elements of the first block that are in front of the row
    uint32_t n_vocab, blocks;
    uint32_t from, to;
    const uint32_t* mask;
};

// The mask's bits of block b's elements (of those in front of the row too: of no meaning).
template <uint32_t N>
__device__ __forceinline__ uint32_t mask_of(const Columns& c, uint32_t b)
{
    const int32_t first = (int32_t)(b * N) - (int32_t)c.before;
    const uint32_t at = first < 0 ? 0u : (uint32_t)first, word = at / 32u, last = (c.n_vocab - 1u) / 32u;
    const uint32_t bits = __funnelshift_r(__ldg(c.mask + min(word, last)), __ldg(c.mask + min(word + 1u, last)), at & 31u);
    return first < 0 ? bits << -first : bits;
}

// Which of block b's elements are the row's own, of those that the mask allows.
template <uint32_t N>
__device__ __forceinline__ uint32_t there_of(const Columns& c, uint32_t b, uint32_t allowed)
{
    const int32_t first = (int32_t)(b * N) - (int32_t)c.before;
    uint32_t there = allowed & ((1u << N) - 1u);
    if (first < 0)
        there &= ~0u << -first;
    if (first + (int32_t)N > (int32_t)c.n_vocab)
        there &= first >= (int32_t)c.n_vocab ? 0u : (1u << (c.n_vocab - first)) - 1u;
    return there;
}

template <typename T>
__device__ __forceinline__ void take_out(uint32_t (&w)[4], uint32_t there)
{
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        w[i] = Words<T>::without(w[i], there >> (i * Words<T>::each));
}

// Block b of a row as it is, for what is done rarely.
template <typename T, bool Mask>
__device__ __forceinline__ uint32_t read_block(const Columns& c, uint32_t b, uint32_t (&w)[4])
{
    const uint4 x = c.base[b];
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    const uint32_t there = there_of<4 * Words<T>::each>(c, b, Mask ? mask_of<4 * Words<T>::each>(c, b) : ~0u);
    take_out<T>(w, there);
    return there;
}

// A thread's logits of a tile. Those below `least`, -inf, NaN and what is masked are taken for it, before they become floats where two
// of them are in a word: they weigh nothing then, and nothing times their exponent is not NaN, as long as the largest is far
// enough above, and exponents are of a size at which a shift is rounded by less than 2^6 (reachable() below says whether they are; if not the
// row's sums are formed again).
template <typename T, uint32_t Blocks>
__device__ __forceinline__ void add(Sums<float>& s, const uint32_t (&w)[Blocks][4], float c, float most)
{
    if (!(most > Words<T>::least)) // nothing that weighs anything
        return;
    const float shift = most * c;
    if (shift > s.shift) {
        const float d = fmaxf(s.shift - shift, kLeast), f = ex2_approx(d);
        s.wd = f * (s.wd + d * s.w);
        s.w *= f;
        s.shift = shift;
    }
    const float2 c2 = make_float2(c, c), minus = make_float2(-s.shift, -s.shift);
    float2 w2 = make_float2(0.0f, 0.0f), d2 = w2;
#pragma unroll
    for (uint32_t j = 0; j < Blocks; ++j) {
        uint32_t y[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            y[i] = Words<T>::larger(w[j][i], Words<T>::of_least());
#pragma unroll
        for (uint32_t i = 0; i < 4; i += 2 / Words<T>::each) {
            const float2 d = fma2(Words<T>::pair(y + i), c2, minus);
            const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
            w2 = add2(w2, e);
            d2 = fma2(e, d, d2);
        }
    }
    s.w += w2.x + w2.y;
    s.wd += d2.x + d2.y;
}

// Are sums formed so right, of a row whose largest is `most`?
template <typename T>
__device__ __forceinline__ bool reachable(float most, float c)
{
    return (most - Words<T>::least) * c >= 200.0f && fabsf(Words<T>::least * c) < 0x1p30f && fabsf(most * c) < 0x1p30f;
}

// Leaves the k largest of the list's n keys (n <= kListCap) at its front, in no order, by all threads; returns how many there are.
__device__ uint32_t keep_best(Shared& s, uint32_t n, uint32_t k)
{
    const uint32_t tid = threadIdx.x;
    __syncthreads();
    if (n <= k)
        return n;
    Key at = 0; // the k-th largest: keys are distinct
    for (int bit = 63; bit >= 0; --bit) {
        const Key want = at | (1ull << bit);
        uint32_t count = 0;
        for (uint32_t i = tid; i < n; i += kThreads)
            count += s.list[i] >= want;
        s.largest[tid] = __uint_as_float(count);
        __syncthreads();
        uint32_t all = 0;
        for (uint32_t i = tid & 31u; i < kThreads; i += 32u)
            all += __float_as_uint(s.largest[i]);
        all = __reduce_add_sync(~0u, all);
        if (all >= k)
            at = want;
        __syncthreads();
    }
    constexpr uint32_t each = (kListCap + kThreads - 1) / kThreads;
    Key mine[each];
#pragma unroll
    for (uint32_t j = 0; j < each; ++j) {
        const uint32_t i = tid + j * kThreads;
        mine[j] = i < n ? s.list[i] : 0;
    }
    if (tid == 0)
        s.n = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < each; ++j)
        if (mine[j] && mine[j] >= at)
            s.list[atomicAdd(&s.n, 1u)] = mine[j];
    __syncthreads();
    return k;
}

// How many of n keys are above one.
__device__ __forceinline__ uint32_t above(const Key* list, uint32_t n, Key mine)
{
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < n; ++i)
        rank += list[i] > mine;
    return rank;
}

// The k largest of the list's first n keys in order, into `best`: each ranked against the others, kRankMax of them at a time. The
// list is whole; behind it all threads see what is in `best`.
__device__ void rank_best(Shared& s, uint32_t n, uint32_t k)
{
    const uint32_t tid = threadIdx.x;
    if (n > 2u * kRankMax)
        n = keep_best(s, n, k);
    uint32_t have = min(n, kRankMax); // ranked so far
    if (tid < have) {
        const Key mine = s.list[tid];
        const uint32_t rank = above(s.list, have, mine);
        if (rank < k)
            s.best[rank] = mine;
    }
    __syncthreads();
    for (uint32_t at = have; at < n;) {
        have = min(have, k);
        const uint32_t some = min(n - at, kRankMax - have), m = have + some;
        const Key mine = tid < have ? s.best[tid] : tid < m ? s.list[at + tid - have] : 0;
        if (tid < m)
            s.ranked[tid] = mine;
        __syncthreads();
        if (tid < m) {
            const uint32_t rank = above(s.ranked, m, mine);
            if (rank < k)
                s.best[rank] = mine;
        }
        __syncthreads();
        have = m;
        at += some;
    }
}

// The same by one warp, of at most kWarpKeys.
__device__ __forceinline__ void rank_by_warp(const Key* list, uint32_t n, uint32_t k, Key* best)
{
    for (uint32_t j = threadIdx.x & 31u; j < n; j += 32u) {
        const Key mine = list[j];
        const uint32_t rank = mine ? above(list, n, mine) : k; // (0 is none)
        if (rank < k)
            best[rank] = mine;
    }
    __syncwarp();
}

// Puts a block's logits above the line into the list.
template <typename T>
__device__ __forceinline__ void put(Shared& s, const Columns& c, uint32_t b, const uint32_t (&w)[4], float line)
{
    constexpr uint32_t each = Words<T>::each;
#pragma unroll
    for (uint32_t i = 0; i < 4u * each; ++i) {
        const float x = Words<T>::value(w[i / each], i % each);
        if (x > line)
            s.list[atomicAdd(&s.n, 1u)] = make_key(x, b * 4u * each - c.before + i);
    }
}

template <typename T, bool Mask>
__global__ void __launch_bounds__(kThreads, 5) logprob_kernel(const mk_logprob_rows r, const LogprobOut o)
{
    constexpr uint32_t N = 4 * Words<T>::each, kTile = kThreads * kTileVecs;
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t slices = cluster.num_blocks(), slice = cluster.block_rank(), row = blockIdx.x / slices;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, k = r.n_top ? r.n_top : 1u;
    griddep_launch_dependents();
    if (tid == 0) {
        s.n = 0;
        s.allowed = 0;
        s.line = ~0u;
    }
    __syncwarp();
    if (slices > 1)
        cluster_arrive();
    griddep_wait();
    Columns c;
    const T* x0 = static_cast<const T*>(r.logits) + (size_t)row * r.ld;
    c.before = (uint32_t)((reinterpret_cast<uintptr_t>(x0) & 15u) / sizeof(T));
    c.base = reinterpret_cast<const uint4*>(x0 - c.before);
    c.n_vocab = r.n_vocab;
    c.mask = Mask ? r.mask + (size_t)row * r.mask_ld : nullptr;
    c.blocks = (c.before + r.n_vocab + N - 1) / N;
    const uint32_t share = (c.blocks + slices - 1u) >> (31 - __clz((int)slices)); // (a power of two)
    c.from = min(c.blocks, slice * share);
    c.to = min(c.blocks, c.from + share);
    // what is asked of the row, early: two reads one behind the other
    const bool asks = slice == 0 && o.logprob && tid < r.n_given;
    const uint32_t asked = asks ? (uint32_t)r.tokens[(size_t)row * r.n_given + tid] : ~0u;
    const float t = r.temperature ? __ldg(r.temperature + row) : r.temperature_all;
    const bool greedy = !(t > 1e-30f && t < 1e30f);
    const float scale = greedy ? 1.0f : 1.44269504088896340736f / t;

    Sums<float> sums{-INFINITY, 0.0f, 0.0f};
    uint32_t any = 0, tile = 0, turn = 1, line_key = 0;
    float most = -INFINITY;
    const T asked_x = asked < r.n_vocab ? x0[asked] : T(0.0f);
    __syncthreads();
#pragma unroll 1
    for (uint32_t b0 = c.from; b0 < c.to; b0 += kTile, ++tile) {
        uint32_t w[kTileVecs][4], top = Words<T>::none;
        const uint4* p = c.base + b0 + tid;
        if (!Mask && b0 && b0 + kTile <= c.to && b0 + kTile < c.blocks) { // all of it inside the row
#pragma unroll
            for (uint32_t j = 0; j < kTileVecs; ++j) {
                const uint4 x = __ldcs(p + j * kThreads);
                w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
            }
        } else {
            uint32_t there[kTileVecs];
#pragma unroll
            for (uint32_t j = 0; j < kTileVecs; ++j) {
                const uint32_t b = b0 + j * kThreads + tid;
                const uint4 x = b < c.to ? __ldcs(p + j * kThreads) : make_uint4(0, 0, 0, 0);
                there[j] = b >= c.to ? 0u : Mask ? mask_of<N>(c, b) : ~0u;
                w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
            }
#pragma unroll
            for (uint32_t j = 0; j < kTileVecs; ++j) {
                there[j] = there_of<N>(c, b0 + j * kThreads + tid, there[j]);
                any |= there[j];
                take_out<T>(w[j], there[j]);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kTileVecs; ++j)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                top = Words<T>::larger(top, w[j][i]);
        const float here = Words<T>::largest(top);
        if (tile == 0 || tile == turn) { // all threads are here
            if (tile == 0) { // the line starts from the largest of groups of eight threads or, for many alternatives, of each thread
                float group = here;
                if (k <= 8u) {
#pragma unroll
                    for (uint32_t d = 1; d < 8; d <<= 1)
                        group = fmaxf(group, __shfl_xor_sync(~0u, group, d));
                }
                if (k > 8u || tid % 8u == 0)
                    s.largest[k > 8u ? tid : tid / 8u] = group;
                __syncthreads();
                const uint32_t groups = k > 8u ? kThreads : kThreads / 8;
                if (tid < groups) {
                    const float4* all = reinterpret_cast<const float4*>(s.largest);
                    const float mine = s.largest[tid];
                    uint32_t rank = 0;
#pragma unroll 4
                    for (uint32_t i = 0; i < groups / 4; ++i) {
                        const float4 x = all[i];
                        rank += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
                    }
                    __syncwarp();
                    const uint32_t least = __reduce_min_sync(~0u, rank < k ? order_key(mine) : ~0u); // of those that have fewer than k above them
                    if (lane == 0)
                        atomicMin(&s.line, least);
                }
                __syncthreads();
            } else { // and goes up to the k-th largest of what is in the list
                turn *= 2u;
                __syncthreads();
                const uint32_t n = s.n;
                if (tid == 0)
                    s.line_next = ~0u;
                __syncthreads();
                if (n >= k && n <= kThreads && tid < ((n + 31u) & ~31u)) {
                    const uint32_t mine = tid < n ? (uint32_t)(s.list[tid] >> 32) : 0u;
                    const uint32_t* x = reinterpret_cast<const uint32_t*>(s.list) + 1; // the keys' upper words
                    uint32_t rank = 0;
#pragma unroll 4
                    for (uint32_t i = 0; i < n; ++i)
                        rank += x[2u * i] > mine;
                    __syncwarp();
                    const uint32_t least = __reduce_min_sync(~0u, rank < k && tid < n ? mine : ~0u);
                    if (lane == 0)
                        atomicMin(&s.line_next, least);
                }
                __syncthreads();
                if (n >= k && n <= kThreads)
                    line_key = max(line_key, s.line_next);
            }
            if (tile == 0)
                line_key = s.line;
        }
        const float line = key_to_float(line_key);
        // (the line may be a number of this list's own that came behind an equal one: those on it go in as well)
        // A thread that has such a logit is rare: its blocks are handed to the warp, an element or less to each lane.
        uint32_t who = __ballot_sync(~0u, here >= line && here > -INFINITY);
        while (who) {
            const uint32_t from = __ffs(who) - 1;
            who &= who - 1u;
            if (lane == from) {
#pragma unroll
                for (uint32_t j = 0; j < kTileVecs; ++j)
                    s.handed[tid / 32u][j] = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
            }
            __syncwarp();
            if (lane < kTileVecs * N) {
                const float x = (float)reinterpret_cast<const T*>(s.handed[tid / 32u])[lane];
                if (x >= line && x > -INFINITY) {
                    const uint32_t at = atomicAdd(&s.n, 1u);
                    if (at < kListCap)
                        s.list[at] = make_key(x, (b0 + lane / N * kThreads + tid - lane + from) * N - c.before + lane % N);
                }
            }
            __syncwarp();
        }
        most = fmaxf(most, here);
        add<T, kTileVecs>(sums, w, scale, here);
    }
    if (Mask && any)
        s.allowed = 1;
    __syncwarp();
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        sums = join(sums, Sums<float>{__shfl_xor_sync(~0u, sums.shift, d), __shfl_xor_sync(~0u, sums.w, d), __shfl_xor_sync(~0u, sums.wd, d)});
        most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    }
    if (lane == 0) {
        s.warp[tid / 32u] = sums;
        s.warp_most[tid / 32u] = most;
    }
    __syncthreads();
    most = s.warp_most[lane % kWarps];
#pragma unroll
    for (uint32_t d = kWarps / 2; d; d >>= 1)
        most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    uint32_t n = s.n;
    if (n > kListCap) { // read again, piece by piece, with the best of what came before
        uint32_t have = 0;
        float line = -INFINITY;
        __syncthreads();
        for (uint32_t b0 = c.from; b0 < c.to; b0 += kThreads) {
            if (tid == 0)
                s.n = have;
            __syncthreads();
            const uint32_t b = b0 + tid;
            if (b < c.to) {
                uint32_t w[4];
                read_block<T, Mask>(c, b, w);
                put<T>(s, c, b, w, line); // (an equal one comes behind k that are as large; a piece has room)
            }
            __syncthreads();
            const uint32_t now = s.n;
            if (now == have)
                continue;
            have = keep_best(s, now, k);
            if (have == k) {
                if (tid < 32u) {
                    float least = INFINITY;
                    for (uint32_t i = lane; i < k; i += 32u)
                        least = fminf(least, key_x(s.list[i]));
#pragma unroll
                    for (uint32_t d = 16; d; d >>= 1)
                        least = fminf(least, __shfl_xor_sync(~0u, least, d));
                    __syncwarp();
                    if (lane == 0)
                        s.line = order_key(least);
                }
                __syncthreads();
                line = key_to_float(s.line);
            }
        }
        n = have;
    }
    uint32_t n_best = min(n, k);
    if (n > kWarpKeys)
        rank_best(s, n, k);
    else if (tid < 32u)
        rank_by_warp(s.list, n, k, s.best);
    Sums<double> all{-1e300, 0.0f, 0.0f};
    if (n_best && !greedy && most != INFINITY && !reachable<T>(most, scale)) { // a row of the type's lowest value, as masks write it: x - most first
        float w = 0.0f, wd = 0.0f;
        for (uint32_t b = c.from + tid; b < c.to; b += kThreads) {
            uint32_t y[4];
            read_block<T, Mask>(c, b, y);
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const float d = fmaxf((Words<T>::value(y[i / Words<T>::each], i % Words<T>::each) - most) * scale, kLeast), e = ex2_approx(d);
                w += e;
                wd += e * d;
            }
        }
        __syncwarp();
#pragma unroll
        for (uint32_t d = 16; d; d >>= 1) {
            w += __shfl_xor_sync(~0u, w, d);
            wd += __shfl_xor_sync(~0u, wd, d);
        }
        if (lane == 0)
            s.warp[tid / 32u] = Sums<float>{0.0f, w, wd};
        __syncthreads();
        all.shift = (double)most * (double)scale;
        for (uint32_t i = 0; i < kWarps; ++i) {
            all.w += s.warp[i].w;
            all.wd += s.warp[i].wd;
        }
    } else if (n_best) {
        __syncwarp();
        Sums<float> x = s.warp[lane % kWarps];
#pragma unroll
        for (uint32_t d = kWarps / 2; d; d >>= 1)
            x = join(x, Sums<float>{__shfl_xor_sync(~0u, x.shift, d), __shfl_xor_sync(~0u, x.w, d), __shfl_xor_sync(~0u, x.wd, d)});
        all = Sums<double>{(double)x.shift, x.w, x.wd};
    }
    uint32_t allowed = s.allowed;
    // from here on the first warp is enough, unless there are many keys or tokens
    if (slices > 1) { // each slice leaves what it has with the first one
        __syncwarp();
        cluster_wait(); // all of them run
        if (tid < 32u) {
            Shared* first = cluster.map_shared_rank(&s, 0);
            for (uint32_t i = lane; i < k; i += 32u)
                first->of_slices[slice * k + i] = i < n_best ? s.best[i] : 0;
            if (lane == 0) {
                first->slice_sums[slice] = all;
                first->slice_most[slice] = most;
                first->slice_has[slice] = n_best | (allowed ? 0x100u : 0u);
            }
        }
        __syncwarp();
        cluster_arrive();
        if (slice)
            return;
        cluster_wait();
        all = Sums<double>{-1e300, 0.0f, 0.0f};
        most = -INFINITY;
        uint32_t has = 0;
        if (lane < slices) {
            all = s.slice_sums[lane];
            most = s.slice_most[lane];
            has = s.slice_has[lane];
        }
        __syncwarp();
#pragma unroll
        for (uint32_t d = kMaxCluster / 2; d; d >>= 1) {
            all = join(all, Sums<double>{__shfl_xor_sync(~0u, all.shift, d), __shfl_xor_sync(~0u, all.w, d), __shfl_xor_sync(~0u, all.wd, d)});
            most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
        }
        // (the upper lanes' are those of none)
        all = Sums<double>{__shfl_sync(~0u, all.shift, 0), __shfl_sync(~0u, all.w, 0), __shfl_sync(~0u, all.wd, 0)};
        most = __shfl_sync(~0u, most, 0);
        n_best = min(k, __reduce_add_sync(~0u, has & 0xffu));
        allowed = __any_sync(~0u, has & 0x100u);
        const uint32_t keys = slices * k; // distinct but for those that are none, 0
        if (keys <= kWarpKeys) {
            if (tid < 32u)
                rank_by_warp(s.of_slices, keys, k, s.best);
        } else {
            for (uint32_t i = tid; i < keys; i += kThreads) {
                const Key key = s.of_slices[i];
                const uint32_t rank = key ? above(s.of_slices, keys, key) : k;
                if (rank < k)
                    s.best[rank] = key;
            }
        }
    }
    if (k <= 32u && r.n_given <= 32u && (slices == 1 ? n : slices * k) <= kWarpKeys) {
        if (tid >= 32u)
            return;
        __syncwarp();
    } else {
        __syncthreads();
    }
    // one token alone: greedy, an infinite logit, or logits that are so far from one another that none but the largest weighs anything
    const bool one = n_best && (greedy || most == INFINITY || !(all.w > 0.0f));
    const float log2_sum = one ? 0.0f : log2f(all.w);
    constexpr float ln2 = 0.693147180559945309417f;
    // ln of the sum of e^((x - most) / t): the shift is that of the largest but for its rounding
    const float ln_sum = one || n_best == 0 ? 0.0f : (float)(0.693147180559945309417 * ((double)log2_sum - ((double)most * (double)scale - all.shift)));
    auto logprob = [&](float x, uint32_t id) {
        if (n_best == 0 || !(x > -INFINITY)) // (NaN too)
            return -INFINITY;
        if (one)
            return id == key_id(s.best[0]) ? 0.0f : -INFINITY;
        return __fdiv_rn(x - most, t) - ln_sum;
    };
    if (o.logprob)
        for (uint32_t i = tid; i < r.n_given; i += kThreads) {
            const uint32_t id = i == tid ? asked : (uint32_t)r.tokens[(size_t)row * r.n_given + i];
            float y = 0.0f; // of no token
            if (id < r.n_vocab) {
                const bool there = !Mask || (__ldg(c.mask + id / 32u) >> (id & 31u)) & 1u;
                y = logprob(!there ? -INFINITY : i == tid ? (float)asked_x : (float)x0[id], id);
            }
            o.logprob[(size_t)row * r.n_given + i] = y;
        }
    if (tid < r.n_top) {
        const Key key = tid < n_best && !(one && tid) ? s.best[tid] : 0;
        if (o.top_ids)
            o.top_ids[(size_t)row * r.n_top + tid] = key ? (int32_t)key_id(key) : -1;
        if (o.top_logprob)
            o.top_logprob[(size_t)row * r.n_top + tid] = key ? logprob(key_x(key), key_id(key)) : -INFINITY;
    }
    if (tid == 0) {
        if (o.entropy)
            o.entropy[row] = one || n_best == 0 ? 0.0f : ln2 * (log2_sum - all.wd / all.w);
        if (o.flags)
            o.flags[row] = n_best ? 0u : MK_FLAG_NO_CANDIDATE | (Mask && !allowed ? MK_FLAG_ALL_MASKED : 0u);
    }
}

template <typename T, bool Mask>
cudaError_t launch(const mk_logprob_rows& r, const LogprobOut& o, cudaStream_t stream)
{
    uint32_t slices = 1;
    while (slices < kMaxCluster && r.rows * slices < 148u * 3u && r.n_vocab / (2u * slices) >= 2048u)
        slices *= 2u;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = set_once(done, logprob_kernel<T, Mask>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(r.rows * slices);
    c.blockDim = dim3(kThreads);
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = slices;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    c.attrs = attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, logprob_kernel<T, Mask>, r, o);
}

} // namespace

cudaError_t launch_token_logprobs(const mk_logprob_rows& r, const LogprobOut& o, cudaStream_t stream)
{
    switch (r.type) {
    case MK_FP32: return r.mask ? launch<float, true>(r, o, stream) : launch<float, false>(r, o, stream);
    case MK_BF16: return r.mask ? launch<__nv_bfloat16, true>(r, o, stream) : launch<__nv_bfloat16, false>(r, o, stream);
    default: return r.mask ? launch<__half, true>(r, o, stream) : launch<__half, false>(r, o, stream);
    }
}

} // namespace mk
