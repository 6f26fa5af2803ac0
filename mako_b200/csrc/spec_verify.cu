// Verification of a speculative round against whole distributions (mk_spec_verify in include/mako_b200.h), two launches.
//
// The first reads rows, two CTAs on every SM that take their work from a common counter: a slice of a position's two rows, the
// target's and the drafter's, through a ring of 16 KB tiles (bulk copies by one warp, eight warps behind it). What bounds it is that
// reading. Work comes position by position, the first one of all sequences before the second one, and the last CTA to finish a
// position decides its draft; a slice of a sequence whose round has ended by then is passed over, so that most of the rows behind a
// refused draft, about half of all as drafters go, are never read. (Which ones are read depends on timing, what comes out does not.
// As one cluster per sequence that walks its positions in turn, the chain of reads, exchanges and decisions took 5 us a position; as
// a CTA per slice, the CTAs spent two thirds of their lives on starting and ending.)
// Each thread keeps a running maximum and sum of exp2((x - max) log2(e) / T) in fp32, good to about 1e-6; a decision nearer than
// kNear is left to the second launch. 64 sequences of four drafts, 129280 columns in fp32: 55 us for 234 MB.
//
// The second draws, a cluster of CTAs per sequence. In a vocabulary's running sum every token lies next to others, so weights and
// sums are in 64 bits here: exp2 by a table of 16 steps (one row of the banks: no conflicts) and a quartic, error 4e-11. max(0, P - Q)
// wants both rows' whole weights first; instead of a pass for them, the one pass forms A = sum of (p - c q) and B = sum of q over the
// columns where p > c q, with the c = P's / Q's whole weight that the fp32 sums give, beside the exact sums, and A - (exact c - c) B is
// what is drawn from: only columns between the two c, 1e-6 apart, are off, by as much again (rows so alike that this matters are drawn from
// once more, see draw()). The sums by CTA and warp lead to one warp's columns, which the CTA goes over once more, eight a thread. 52 us for
// the same sequences, 16 for a single one: neither the 64-bit pipe (23 operations a column, a quarter of its rate) nor DRAM (65 MB, 17 %)
// bounds it, it waits: 0.44 instructions a cycle from 24 warps an SM of 80 registers, one block of 16 bytes a lane under way, and its few
// steps one behind another.
#include "ptx.cuh"
#include "round_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

constexpr uint32_t kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32, kMaxCluster = 16;
constexpr uint32_t kDrawThreads = 384, kDrawWarps = kDrawThreads / 32;
constexpr uint32_t kTileBlocks = 1024, kTileBytes = 16 * kTileBlocks, kTiles = 6; // of the ring
constexpr uint32_t kScanCtas = 296; // two on each of 148 SMs
constexpr uint32_t kScanThreads = kVerifyThreads + 64; // and a warp that copies, and one that closes pieces of work
constexpr uint32_t kSteps = 16;   // of the table of exp2
constexpr uint32_t kParts = 8;   // of a warp's share of a row
constexpr float kNear = 3e-5f;    // decisions nearer than this, relative, are taken in 64 bits
constexpr float kFew = 1e-30f;    // and those of probabilities of which fp32 may hold few bits or none: ex2_approx ends at 2^-126
constexpr double kLoose = 1e-4, kLittle = 1e-6; // see draw()
constexpr double kSome = 1e-290;   // a weight below this, where the largest is about 1, is none
constexpr double kSteepest = 3e38; // log2(e) / T above this is none of fp32's numbers
constexpr float kHottest = 1e30f;  // a temperature from here on is not one
constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// The columns of 16 bytes, in pairs.
__device__ __forceinline__ void to_pairs(float2 (&x)[2], const uint4& w, float)
{
    x[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    x[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ void to_pairs(float2 (&x)[4], const uint4& w, __nv_bfloat16)
{
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
}
__device__ __forceinline__ void to_pairs(float2 (&x)[4], const uint4& w, __half)
{
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
}

// The largest of the columns of N times 16 bytes, two 16-bit ones at a time.
template <int N>
__device__ __forceinline__ float largest(const uint4 (&w)[N], float)
{
    float top = -kInf;
#pragma unroll
    for (int i = 0; i < N; ++i)
        top = fmaxf(top, fmaxf(fmaxf(__uint_as_float(w[i].x), __uint_as_float(w[i].y)), fmaxf(__uint_as_float(w[i].z), __uint_as_float(w[i].w))));
    return top;
}
template <int N, typename P>
__device__ __forceinline__ float largest_pairs(const uint4 (&w)[N], P)
{
    P top = *reinterpret_cast<const P*>(&w[0].x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t r[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            top = __hmax2(top, *reinterpret_cast<const P*>(&r[e]));
    }
    return fmaxf(to_float(top.x), to_float(top.y));
}
template <int N>
__device__ __forceinline__ float largest(const uint4 (&w)[N], __nv_bfloat16) { return largest_pairs(w, __nv_bfloat162()); }
template <int N>
__device__ __forceinline__ float largest(const uint4 (&w)[N], __half) { return largest_pairs(w, __half2()); }

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    unsigned long long ra, rb, rd;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t cluster_size()
{
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The place of `p`, a shared variable, in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}

__device__ __forceinline__ void put(uint32_t at, double a, double b)
{
    asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at), "d"(a), "d"(b) : "memory");
}

// A maximum m and the sum of 2^(x scale - fl(m scale)): the product rounds once, in the FMA, so that its reference point is
// exact; -inf and 0 where there is none. A row whose reference point is beyond kFar (logits of the type's lowest value, temperatures
// of next to nothing) is weighed in 64 bits, as that point is off by more than a little itself. A part of a row, which lies below the
// row's own largest where that is negative, makes its sum up to kSum: parts beyond that weigh 2^-4096 at most in a row that is not far.
constexpr float kFar = 1e6f, kSum = kFar + 4096.0f;
struct Mass {
    float m, s;
    __device__ void add(const Mass& o, float scale)
    {
        const float top = fmaxf(m, o.m);
        if (fabsf(__fmul_rn(top, scale)) < kSum) { // else nothing yet, or a sum that no one will use
            const float mine = m > -kInf ? s * ex2_approx(__fmul_rn(m, scale) - __fmul_rn(top, scale)) : 0.0f;
            s = mine + (o.m > -kInf ? o.s * ex2_approx(__fmul_rn(o.m, scale) - __fmul_rn(top, scale)) : 0.0f);
        }
        m = top;
    }
};

template <typename T>
struct Row {
    const T* x;
    const uint32_t* mask; // or nullptr
    float t;              // temperature; 0: the largest alone
    float scale;          // log2(e) / t
    double scale64;
    float lowest;         // what is below this weighs 2^-1000, which is nothing, of a row with a maximum
    Mass mass;            // of the whole row
    double sum64;         // its whole weight in the draw's units, of a far() row
    __device__ void temperature(float v)
    {
        t = v > 0.0f && v < kHottest ? v : 0.0f;
        scale64 = t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
        scale = (float)fmin(scale64, kSteepest);
    }
    __device__ void weighed(const Mass& a)
    {
        mass = a;
        lowest = fmaxf((a.m - base()) - 693.0f * t, -3.4e38f);
    }
    __device__ bool none() const { return mass.m == -kInf; }
    __device__ bool off() const { return !(fabsf(__fmul_rn(mass.m, scale)) < kFar) || scale64 > kSteepest; } // the fp32 sums are
    __device__ bool far() const { return !none() && !single() && off(); }
    __device__ float base() const { return off() ? mass.m : 0.0f; }
    __device__ double zero() const { return rint((double)(mass.m - base()) * scale64 * kSteps); }
    // The whole weight where the step of the draw's table next to the largest weighs 1, as good as the fp32 sums are. Those stand on
    // fl(m scale) in units of the fp32 scale, which is off by 2^-25 of itself: 0.03 of a power of two where m scale is 1e6.
    __device__ double whole() const
    {
        if (far())
            return sum64;
        const double d = (((double)__fmul_rn(mass.m, scale) - zero() / kSteps) + (double)mass.m * (scale64 - (double)scale)) * 0.6931471805599453;
        return (double)mass.s * (1.0 + d * (1.0 + d * (1.0 / 2.0 + d * (1.0 / 6.0 + d / 24.0)))); // |d| < 0.1
    }
    // A logit's logarithm of its part. From the fp32 sums, which are off by 1e-7 as fp32 itself is for logarithms of a few units: a
    // kept draft's whole weight in 64 bits would be a pass over its row.
    __device__ float log_part(float x) const
    {
        if (far())
            return (float)(((double)(x - base()) * scale64 - zero() / kSteps) * 0.6931471805599453 - log(sum64));
        return (float)(((double)x * (double)scale - (double)__fmul_rn(mass.m, scale)) * 0.6931471805599453) - logf(mass.s);
    }
    __device__ bool single() const { return t == 0.0f || mass.m == kInf; }
    // A column's logit; what is masked or NaN is -inf.
    __device__ float get(uint32_t i) const
    {
        const bool off = mask && !((__ldg(mask + (i >> 5)) >> (i & 31u)) & 1u);
        return off ? -kInf : fmaxf(to_float(x[i]), -kInf);
    }
};

struct Sums {
    double a, b, p, q;
};

struct Shared {
    double table[kSteps];
    double2 slices[2][kMaxCluster][2]; // what each CTA of the cluster sent, in turns
    Sums warp[kDrawWarps];
    double2 upto[kDrawWarps][kParts]; // A and B of a warp's blocks up to the end of each part of them
    double run[kDrawWarps];
    uint32_t first[kDrawWarps];
    int32_t token;
};

// One CTA's part in a cluster, and the turn of the exchanges.
struct Part {
    uint32_t rank, size, n, turn;
};

// Sends x, the same in the first `size` threads, to every CTA; after it slices[turn] has all.
__device__ __forceinline__ const double2 (*exchange(Shared& s, Part& c, const Sums& x))[2]
{
    const double2(*got)[2] = s.slices[c.turn];
    if (threadIdx.x < c.size) {
        const uint32_t to = in_cta(&s.slices[c.turn][c.rank][0], threadIdx.x);
        put(to, x.a, x.b);
        put(to + 16u, x.p, x.q);
    }
    c.turn ^= 1u;
    cluster_sync();
    return got;
}

// A row as blocks of 16 bytes: block b has the columns b * per - odd on, of which those outside of the row are off.
template <typename T>
struct Blocks {
    static constexpr uint32_t per = 16 / sizeof(T);
    uint32_t odd, count;
    __device__ Blocks(const T* x, uint32_t n)
    {
        odd = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
        count = (n + odd + per - 1u) / per;
    }
    __device__ int32_t column(uint32_t b) const { return (int32_t)(b * per) - (int32_t)odd; }
};

// Which of the `per` columns from i0 on are in the row and allowed, as bits.
template <typename T>
__device__ __forceinline__ uint32_t columns_on(const uint32_t* mask, int32_t i0, uint32_t n)
{
    constexpr uint32_t per = Blocks<T>::per;
    uint32_t on = (1u << per) - 1u;
    if (i0 < 0)
        on &= on << -i0;
    const int32_t left = (int32_t)n - i0;
    if (left < (int32_t)per)
        on = left <= 0 ? 0u : on & ((1u << left) - 1u);
    if (mask && on) {
        const uint32_t lo = __ldg(mask + (max(i0, 0) >> 5)), hi = __ldg(mask + (min(i0 + (int32_t)per - 1, (int32_t)n - 1) >> 5));
        on &= i0 < 0 ? lo << -i0 : __funnelshift_r(lo, hi, (uint32_t)i0 & 31u);
    }
    return on;
}

// A thread's share of a row in the pass for its maximum and sum.
template <typename T>
struct Scan {
    static constexpr int kDeep = kTileBlocks / kVerifyThreads, per = (int)Blocks<T>::per;
    Mass a{-kInf, 0.0f};
    uint32_t at = ~0u; // the first column that holds the maximum, where asked for

    // The thread's blocks of a tile: columns i0 + k * kVerifyThreads * per on, of which `on` (bits, per for each block) count; false:
    // there was a NaN where all of them were to count.
    template <bool Whole>
    __device__ __forceinline__ bool tile(const uint4 (&w)[kDeep], uint32_t on, float scale, bool greedy, int32_t i0)
    {
        float2 x[kDeep][per / 2];
#pragma unroll
        for (int i = 0; i < kDeep; ++i)
            to_pairs(x[i], w[i], T());
        float top = -kInf;
        if (Whole) { // (fmaxf and its like pass over NaN)
            top = largest<kDeep>(w, T());
        } else {
#pragma unroll
            for (int i = 0; i < kDeep; ++i)
#pragma unroll
                for (int e = 0; e < per / 2; ++e) { // what is off or NaN is -inf
                    x[i][e].x = on >> (per * i + 2 * e) & 1u ? fmaxf(x[i][e].x, -kInf) : -kInf;
                    x[i][e].y = on >> (per * i + 2 * e + 1) & 1u ? fmaxf(x[i][e].y, -kInf) : -kInf;
                    top = fmaxf(top, fmaxf(x[i][e].x, x[i][e].y));
                }
        }
        const float m = fmaxf(a.m, top);
        float all = 0.0f;
        const bool near = fabsf(__fmul_rn(m, scale)) < kSum;
        if (near) {
            const float2 by = make_float2(scale, scale), off = make_float2(-__fmul_rn(m, scale), -__fmul_rn(m, scale));
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < kDeep; ++i)
#pragma unroll
                for (int e = 0; e < per / 2; ++e) {
                    const float2 t = fma2(x[i][e], by, off);
                    sum[e & 1] = add2(sum[e & 1], make_float2(ex2_approx(t.x), ex2_approx(t.y)));
                }
            all = (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
            if (Whole && all != all)
                return false;
        } else if (Whole) { // no sum that would show one
            return false;
        }
        if (top > a.m) {
            a.s = a.s == 0.0f || !near ? 0.0f : a.s * ex2_approx(__fmul_rn(a.m, scale) - __fmul_rn(top, scale));
            a.m = top;
            if (greedy || top == kInf) {
#pragma unroll
                for (int i = kDeep - 1; i >= 0; --i)
#pragma unroll
                    for (int e = per - 1; e >= 0; --e)
                        if ((e & 1 ? x[i][e / 2].y : x[i][e / 2].x) == top)
                            at = (uint32_t)(i0 + i * (int)kVerifyThreads * per + e);
            }
        }
        a.s += all;
        return true;
    }
};

// The part of `count` blocks that falls to `rank` of `size`.
__device__ __forceinline__ uint32_t share(uint32_t count, uint32_t rank, uint32_t size) { return (uint32_t)((uint64_t)count * rank / size); }

// The maximum and sum of all lanes' masses, the same bits in every lane; at: the least of those that go with the maximum.
__device__ __forceinline__ Mass warp_merge(Mass a, float scale, uint32_t& at)
{
    float top = a.m;
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    at = __reduce_min_sync(~0u, a.m == top ? at : ~0u);
    float s = 0.0f;
    if (fabsf(__fmul_rn(top, scale)) < kSum && a.s != 0.0f)
        s = a.s * ex2_approx(__fmul_rn(a.m, scale) - __fmul_rn(top, scale));
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        s += __shfl_xor_sync(~0u, s, d);
    return Mass{top, s};
}

enum : uint32_t { kKept = 1, kEnds = 2, kOpen = 3 }; // kOpen: for the second launch to decide

// What a sequence's rows have in common, and where a position's rows lie.
template <typename T>
__device__ __forceinline__ void heat_rows(const mk_spec_rows& r, uint32_t sq, Row<T>& p, Row<T>& q)
{
    const float t = r.temperature ? r.temperature[sq] : r.temperature_all;
    p.temperature(t);
    q.temperature(r.draft_temperature ? r.draft_temperature[sq] : t);
}

template <typename T>
__device__ __forceinline__ void place_rows(const mk_spec_rows& r, uint32_t sq, uint32_t j, bool against, Row<T>& p, Row<T>& q)
{
    const size_t row = (size_t)sq * r.n_pos + j, drow = (size_t)sq * (r.n_pos - 1u) + j;
    p.x = static_cast<const T*>(r.logits) + row * r.ld;
    p.mask = r.mask ? r.mask + row * r.mask_ld : nullptr;
    q.x = against ? static_cast<const T*>(r.draft_logits) + drow * r.draft_ld : nullptr;
    q.mask = r.mask_drafts ? p.mask : nullptr;
}

// P(d) and u Q(d) in fp32, from the rows' masses.
template <typename T>
__device__ __forceinline__ float part_of(const Row<T>& r, float x, uint32_t at, uint32_t d)
{
    return r.none() ? 0.0f : r.single() ? (at == d ? 1.0f : 0.0f) : ex2_approx(fmaf(x, r.scale, -__fmul_rn(r.mass.m, r.scale))) / r.mass.s;
}

// A tile of the ring: what it holds of which row.
struct Tile {
    uint32_t sq, j, slice;
    int32_t column;     // of its first block
    uint32_t blocks;    // 0: there is no more work
    const uint32_t* mask;
    float scale, scale_p; // of its row, and of the target's
    uint32_t what;        // bits of:
};
enum : uint32_t { kDrafters = 1, kFirstTile = 2, kLastTile = 4, kGreedy = 8, kDrafted = 16, kAgainst = 32 };

struct ScanShared {
    uint64_t full[kTiles], empty[kTiles];
    uint64_t there[2], taken[2]; // of what follows
    Tile piece[2];               // the last tile of a piece of work; of no blocks: there are no more
    Tile tile[kTiles];
    Mass mass[2][2][kVerifyWarps]; // two pieces of work in turn; the target's, the drafter's
    uint32_t at[2][2][kVerifyWarps];
    int failed;
};

// Waits, but not for ever: one of two seconds, in any warp, ends all.
__device__ __forceinline__ bool await(int* failed, uint64_t* bar, uint32_t parity)
{
    if (mbar_try(bar, parity))
        return true;
    const long long from = clock64();
    do {
        if (mbar_try(bar, parity))
            return true;
    } while (clock64() - from < (1ll << 32) && !*reinterpret_cast<volatile int*>(failed));
    *reinterpret_cast<volatile int*>(failed) = 1;
    return false;
}

// The copying warp: takes pieces of work, passes over those that are of no use any more, requests the others' tiles.
template <typename T>
__device__ void copy_tiles(const SpecVerifyArgs& a, ScanShared& s, unsigned char* ring)
{
    const mk_spec_rows& r = a.r;
    const uint32_t lane = threadIdx.x & 31u, n = r.n_vocab, n_drafts = r.n_pos - 1u, total = r.n_seq * r.n_pos * a.slices;
    uint32_t slot = 0, parity = 1;
    bool ok = true;
    auto take = [&]() { return lane == 0 ? atomicAdd(a.counter, 1u) : 0u; };
    uint32_t mine = take();
    while (ok) {
        const uint32_t item = __shfl_sync(~0u, mine, 0);
        if (item >= total)
            break;
        mine = take(); // the next one is on its way meanwhile
        const uint32_t slice = item % a.slices, sq = item / a.slices % r.n_seq, j = item / a.slices / r.n_seq;
        const int32_t* drafts = r.drafts + (size_t)sq * n_drafts;
        const uint32_t ended = __ldcg(&a.ended[sq]); // 0, or all ones less the position of the end
        bool over = ended && ~ended < j;
        for (uint32_t i = lane; i < j; i += 32)
            over |= (uint32_t)drafts[i] >= n;
        const int32_t d = j < n_drafts ? drafts[j] : -1;
        Row<T> p, q;
        heat_rows(r, sq, p, q);
        if (__any_sync(~0u, over))
            continue;
        const bool drafted = (uint32_t)d < n, against = drafted && r.draft_logits;
        place_rows(r, sq, j, against, p, q);
        for (uint32_t which = 0; which < (against ? 2u : 1u) && ok; ++which) {
            const Row<T>& row = which ? q : p;
            const Blocks<T> k(row.x, n);
            const uint32_t to = share(k.count, slice + 1u, a.slices);
            for (uint32_t b = share(k.count, slice, a.slices), first = kFirstTile; b < to && ok; b += kTileBlocks, first = 0) {
                if (!(ok = await(&s.failed, &s.empty[slot], parity)))
                    break;
                const uint32_t blocks = min(to - b, kTileBlocks);
                if (lane == 0) {
                    s.tile[slot] = Tile{sq, j, slice, k.column(b), blocks, row.mask, row.scale, p.scale,
                                        which | first | (b + blocks == to ? kLastTile : 0u) | (row.t == 0.0f ? kGreedy : 0u) |
                                            (drafted ? kDrafted : 0u) | (against ? kAgainst : 0u)};
                    mbar_arrive_expect_tx(&s.full[slot], blocks * 16u);
                    bulk_load(ring + slot * kTileBytes, row.x + k.column(b), blocks * 16u, &s.full[slot]);
                }
                if (++slot == kTiles) {
                    slot = 0;
                    parity ^= 1u;
                }
            }
        }
    }
    if (await(&s.failed, &s.empty[slot], parity) && lane == 0) {
        s.tile[slot] = Tile{};
        mbar_arrive(&s.full[slot]);
    }
}

// The end of a piece of work, by one warp: its masses join the position's, which the last piece decides.
template <typename T>
__device__ void close_piece(const SpecVerifyArgs& a, const Tile& z, Mass mp, uint32_t at_p, Mass mq, uint32_t at_q)
{
    const mk_spec_rows& r = a.r;
    const uint32_t lane = threadIdx.x & 31u;
    const bool drafted = z.what & kDrafted, against = z.what & kAgainst;
    mp = warp_merge(mp, z.scale_p, at_p);
    mq = warp_merge(mq, z.scale, at_q);
    const size_t row = (size_t)z.sq * r.n_pos + z.j;
    SpecPart* parts = a.parts + row * a.slices;
    uint32_t before = 0;
    if (lane == 0) {
        parts[z.slice] = SpecPart{mp.m, mp.s, at_p, 0u, mq.m, mq.s, at_q, 0u};
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(&a.tickets[row]) : "memory");
    }
    if (__shfl_sync(~0u, before, 0) != a.slices - 1u)
        return;
    __syncwarp(); // what the first lane's counting made visible to it is so to the others (a shuffle orders no memory)
    Row<T> p, q;
    heat_rows(r, z.sq, p, q);
    place_rows(r, z.sq, z.j, against, p, q);
    uint32_t d = 0;
    float x = 0.0f, y = 0.0f, u = 0.0f;
    if (drafted) {
        d = (uint32_t)r.drafts[(size_t)z.sq * (r.n_pos - 1u) + z.j];
        u = r.u[(size_t)z.sq * (r.n_pos + 1u) + z.j];
        x = p.get(d);
        if (against)
            y = q.get(d);
    }
    mp = mq = Mass{-kInf, 0.0f};
    at_p = at_q = ~0u;
    for (uint32_t k = 0; k < a.slices; k += 32) { // (at most twice, in order)
        Mass vp{-kInf, 0.0f}, vq{-kInf, 0.0f};
        uint32_t fp = ~0u, fq = ~0u;
        if (k + lane < a.slices) {
            const float4* z = reinterpret_cast<const float4*>(&parts[k + lane]);
            const float4 zp = __ldcg(z), zq = __ldcg(z + 1);
            vp = Mass{zp.x, zp.y};
            vq = Mass{zq.x, zq.y};
            fp = __float_as_uint(zp.z);
            fq = __float_as_uint(zq.z);
        }
        vp = warp_merge(vp, p.scale, fp);
        vq = warp_merge(vq, q.scale, fq);
        at_p = vp.m > mp.m ? fp : vp.m == mp.m ? min(at_p, fp) : at_p;
        at_q = vq.m > mq.m ? fq : vq.m == mq.m ? min(at_q, fq) : at_q;
        mp.add(vp, p.scale);
        mq.add(vq, q.scale);
    }
    if (lane != 0)
        return;
    p.mass = mp;
    q.mass = mq;
    uint32_t state = kEnds;
    if (drafted) {
        const float pd = part_of(p, x, at_p, d), lhs = u * (against ? part_of(q, y, at_q, d) : 1.0f);
        const bool soft_q = against && !q.none() && !q.single();
        const float more = fmaxf(lhs, pd);
        if (p.far() || (soft_q && q.far()) || (((!p.none() && !p.single()) || soft_q) && (fabsf(lhs - pd) <= kNear * more || more < kFew)))
            state = kOpen;
        else if (lhs < pd)
            state = kKept;
    }
    a.states[row] = SpecState{mp.m, mp.s, at_p, state, mq.m, mq.s, at_q, 0u};
    if (state == kEnds)
        atomicMax(&a.ended[z.sq], ~z.j);
}

template <typename T>
__global__ void __launch_bounds__(kScanThreads, 2) spec_scan_kernel(const SpecVerifyArgs a)
{
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ ScanShared s;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, w = tid / 32u, n = a.r.n_vocab;
    if (tid == 0) {
        for (uint32_t i = 0; i < kTiles; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], kVerifyWarps);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&s.there[i], kVerifyWarps);
            mbar_init(&s.taken[i], 1);
        }
        s.failed = 0;
        fence_barrier_init();
    }
    __syncthreads();
    griddep_launch_dependents();
    if (w == kVerifyWarps) {
        copy_tiles<T>(a, s, ring);
    } else if (w == kVerifyWarps + 1u) {
        for (uint32_t turn = 0, parity = 0; await(&s.failed, &s.there[turn], parity); parity ^= turn, turn ^= 1u) {
            const Tile z = s.piece[turn];
            if (z.blocks == 0)
                break;
            Mass mp{-kInf, 0.0f}, mq = mp;
            uint32_t at_p = ~0u, at_q = ~0u;
            if (lane < kVerifyWarps) {
                mp = s.mass[turn][0][lane];
                mq = s.mass[turn][1][lane];
                at_p = s.at[turn][0][lane];
                at_q = s.at[turn][1][lane];
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&s.taken[turn]);
            close_piece<T>(a, z, mp, at_p, mq, at_q);
        }
    } else {
        using Part = Scan<T>;
        constexpr int deep = Part::kDeep, per = Part::per;
        constexpr uint32_t all = per * deep == 32 ? ~0u : (1u << (per * deep % 32)) - 1u;
        uint32_t slot = 0, parity = 0, turn = 0, turn_parity = 0;
        Part x, y; // the target's row; the drafter's
        while (await(&s.failed, &s.full[slot], parity)) {
            const Tile z = s.tile[slot];
            const int32_t i0 = z.column + (int32_t)(tid * per);
            uint4 v[deep];
            uint32_t on = all;
            const bool whole = !z.mask && z.blocks == kTileBlocks && z.column >= 0 && z.column + (int32_t)(kTileBlocks * per) <= (int32_t)n;
            if (!whole) {
                on = 0;
#pragma unroll
                for (int i = 0; i < deep; ++i)
                    if (tid + i * kVerifyThreads < z.blocks)
                        on |= columns_on<T>(z.mask, i0 + i * (int)kVerifyThreads * per, n) << (per * i);
            }
            const uint4* tile = reinterpret_cast<const uint4*>(ring + slot * kTileBytes);
#pragma unroll
            for (int i = 0; i < deep; ++i)
                v[i] = whole || tid + i * kVerifyThreads < z.blocks ? tile[tid + i * kVerifyThreads] : make_uint4(0u, 0u, 0u, 0u);
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&s.empty[slot]);
            if (++slot == kTiles) {
                slot = 0;
                parity ^= 1u;
            }
            if (z.what & kFirstTile) {
                if (z.what & kDrafters)
                    y = x;
                x = Part();
            }
            const bool greedy = z.what & kGreedy;
            if (!(on == all && x.template tile<true>(v, on, z.scale, greedy, i0)) && on)
                x.template tile<false>(v, on, z.scale, greedy, i0);
            if (z.blocks != 0 && (!(z.what & kLastTile) || !(z.what & kDrafters) != !(z.what & kAgainst)))
                continue;
            // the piece's end: x is the last of its rows, y the one before
            const bool against = z.what & kAgainst;
            Mass mp = against ? y.a : x.a, mq = against ? x.a : Mass{-kInf, 0.0f};
            uint32_t at_p = against ? y.at : x.at, at_q = against ? x.at : ~0u;
            mp = warp_merge(mp, z.scale_p, at_p);
            mq = warp_merge(mq, z.scale, at_q);
            if (!await(&s.failed, &s.taken[turn], turn_parity ^ 1u))
                break;
            if (lane == 0) {
                s.mass[turn][0][w] = mp;
                s.mass[turn][1][w] = mq;
                s.at[turn][0][w] = at_p;
                s.at[turn][1][w] = at_q;
                if (w == 0)
                    s.piece[turn] = z;
                mbar_arrive(&s.there[turn]);
            }
            if (z.blocks == 0)
                break;
            turn ^= 1u;
            turn_parity ^= turn == 0;
        }
    }
    __syncthreads();
    if (s.failed && tid == 0) // never seen: the copies in flight end within this; the calls of this handle say what happened
        for (int i = 0; i < 2000; ++i)
            __nanosleep(1000);
    if (s.failed && tid == 0)
        atomicExch(a.failed, 1u);
}

// A row as the draw sees it.
template <typename T>
struct Weigh {
    const T* x;
    const uint32_t* mask;
    float lowest, base; // base: what is taken off every column: nothing, or of a far() row the maximum, which is exact for all that weigh
    int32_t zero;       // the step that weighs 1, next to the maximum's
    double steps;
    __device__ explicit Weigh(const Row<T>& r) : x(r.x), mask(r.mask), lowest(r.lowest), base(r.base()), steps(r.scale64 * kSteps)
    {
        zero = (int32_t)r.zero();
    }
};

// An entry of the table, which lies in shared memory at `table` (as a generic load it took four times as long).
__device__ __forceinline__ double entry(uint32_t table, uint32_t i)
{
    double y;
    asm("ld.shared.f64 %0, [%1];" : "=d"(y) : "r"(table + 8u * i));
    return y;
}

// Weights in 64 bits of columns x of the row, in units of the step next to the maximum's: 2^(k/16) from the table times a quartic
// of the rest r, |r| <= 1/32 of a power: (r ln2)^5 / 120 = 4e-11 at most, of either sign. Fine: two terms more, (r ln2)^7 / 5040 = 5e-16.
// Step by step for all of them, so that their operations stand between one another.
template <bool Fine, int N, typename T>
__device__ __forceinline__ void weights64(const Weigh<T>& row, const float (&x)[N], double (&w)[N], uint32_t table)
{
    constexpr double ln2 = 0.6931471805599453 / kSteps;
    const double shift = 6755399441055744.0; // 1.5 * 2^52: a sum's low bits are its other part to the nearest whole
    double d[N], r[N], y[N];
    uint32_t n[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        d[i] = (double)fmaxf(x[i] - row.base, row.lowest);
#pragma unroll
    for (int i = 0; i < N; ++i)
        r[i] = fma(d[i], row.steps, shift);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        n[i] = (uint32_t)(__double2loint(r[i]) - row.zero);
        y[i] = entry(table, n[i] & (kSteps - 1u));
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        r[i] = shift - r[i];
#pragma unroll
    for (int i = 0; i < N; ++i)
        r[i] = fma(d[i], row.steps, r[i]);
    if (Fine) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            w[i] = fma(ln2 * ln2 * ln2 * ln2 * ln2 * ln2 / 720.0, r[i], ln2 * ln2 * ln2 * ln2 * ln2 / 120.0);
#pragma unroll
        for (int i = 0; i < N; ++i)
            w[i] = fma(w[i], r[i], ln2 * ln2 * ln2 * ln2 / 24.0);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        w[i] = fma(Fine ? w[i] : ln2 * ln2 * ln2 * ln2 / 24.0, r[i], ln2 * ln2 * ln2 / 6.0);
#pragma unroll
    for (int i = 0; i < N; ++i)
        w[i] = fma(w[i], r[i], ln2 * ln2 / 2.0);
#pragma unroll
    for (int i = 0; i < N; ++i)
        w[i] = fma(w[i], r[i], ln2);
#pragma unroll
    for (int i = 0; i < N; ++i)
        w[i] *= r[i];
#pragma unroll
    for (int i = 0; i < N; ++i)
        w[i] = fma(y[i], w[i], y[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) // the power of two
        w[i] = __hiloint2double(__double2hiint(w[i]) + (int)((n[i] & ~(kSteps - 1u)) << 16), __double2loint(w[i]));
}
static_assert(kSteps == 16, "four bits of steps, then the power of two, sixteen places below a double's exponent");

template <typename T>
__device__ __forceinline__ double weight_of(const Row<T>& row, uint32_t i, uint32_t table)
{
    const float x[1] = {row.get(i)};
    double w[1];
    weights64<false>(Weigh<T>(row), x, w, table);
    return w[0] > kSome ? w[0] : 0.0;
}

// x where d = p - c q is above 2^-48 p, else 0; no branch, no comparison of 64 bits. Less than that is what roundings leave of columns that
// weigh the same in P and Q, and would be drawn from where little else is left.
__device__ __forceinline__ double if_more(double x, double d, double p)
{
    const int keep = __double2hiint(d) > __double2hiint(p) - (48 << 20) ? -1 : 0;
    return __hiloint2double(__double2hiint(x) & keep, __double2loint(x) & keep);
}

// What a draw draws from, in units of P's weights: of column i p - c q where that is above 0; q none: p.
template <typename T>
struct Rest {
    Weigh<T> p, q;
    bool against;
    uint32_t without; // column that weighs nothing, or ~0
    double c;
};

// A block of the row, as it lies there: no column of it is left out, and none outside of the row's own 16-byte blocks is read.
template <typename T>
__device__ __forceinline__ uint4 load_block(const Weigh<T>& r, int32_t i0, uint32_t n, bool aligned)
{
    if (aligned)
        return __ldg(reinterpret_cast<const uint4*>(r.x + i0));
    union {
        uint4 w;
        T x[Blocks<T>::per];
    } y;
#pragma unroll
    for (int e = 0; e < (int)Blocks<T>::per; ++e)
        y.x[e] = r.x[min(max(i0 + e, 0), (int32_t)n - 1)];
    return y.w;
}

// Weights of a block's columns of both rows, and f(column's place in the block, p, q) of each. Plain: all columns count.
template <typename T, bool Against, bool Plain, bool Fine, typename F>
__device__ __forceinline__ void each_weight(const Rest<T>& rest, int32_t i0, uint32_t n, const uint4& wp, const uint4& wq,
                                            uint32_t table, F f)
{
    constexpr int per = (int)Blocks<T>::per;
    float2 x[per / 2], y[per / 2];
    to_pairs(x, wp, T());
    if (Against)
        to_pairs(y, wq, T());
    uint32_t on_p = ~0u, on_q = ~0u;
    if (!Plain) {
        on_p = columns_on<T>(rest.p.mask, i0, n);
        if (Against)
            on_q = columns_on<T>(rest.q.mask, i0, n);
    } else if (i0 < 0 || i0 + per > (int32_t)n) { // the row's first or last block
#pragma unroll
        for (int e = 0; e < per; ++e)
            if (i0 + e < 0 || i0 + e >= (int32_t)n) {
                (e & 1 ? x[e / 2].y : x[e / 2].x) = -kInf;
                if (Against)
                    (e & 1 ? y[e / 2].y : y[e / 2].x) = -kInf;
            }
    }
    const uint32_t without = rest.without - (uint32_t)i0;
    // four columns at a time, both rows' together
#pragma unroll
    for (int at = 0; at < per; at += 4) {
        float u[4], v[4];
        double p[4], q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = at + i;
            u[i] = e & 1 ? x[e / 2].y : x[e / 2].x;
            v[i] = Against ? (e & 1 ? y[e / 2].y : y[e / 2].x) : 0.0f;
            if (!Plain) {
                u[i] = on_p >> e & 1u ? u[i] : -kInf;
                v[i] = on_q >> e & 1u ? v[i] : -kInf;
            }
            if (!Against)
                u[i] = without == (uint32_t)e ? -kInf : u[i];
            q[i] = 0.0;
        }
        weights64<Fine>(rest.p, u, p, table);
        if (Against)
            weights64<Fine>(rest.q, v, q, table);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f(at + i, p[i], q[i]);
    }
}

// A warp's share of the CTA's share of a row's blocks, and the blocks of each of its parts.
struct Share {
    uint32_t b0, b1, part;
    __device__ Share(uint32_t count, const Part& c, uint32_t w)
    {
        const uint32_t from = share(count, c.rank, c.size), to = share(count, c.rank + 1u, c.size);
        b0 = from + share(to - from, w, kDrawWarps);
        b1 = from + share(to - from, w + 1u, kDrawWarps);
        part = ((b1 - b0 + kRound - 1u) / kRound + kParts - 1u) / kParts * kRound;
    }
    static constexpr uint32_t kDeep = 1, kRound = 32u * kDeep; // blocks of a lane, and of a warp, under way at a time
};

// The sums over the CTA's share of the row, by warp in s.warp, by its parts in s.upto, and of the CTA: A and B of what is drawn
// from, whole weights.
template <typename T, bool Against, bool Plain, bool Fine>
__device__ __noinline__ Sums sweep_rows(const Rest<T> rest, Shared& s, const Part c)
{
    constexpr int deep = Share::kDeep;
    const uint32_t table = smem_u32(s.table), lane = threadIdx.x & 31u, w = threadIdx.x / 32u, n = c.n;
    const Blocks<T> k(rest.p.x, n);
    const Share mine(k.count, c, w);
    const bool aligned = Plain || (reinterpret_cast<uintptr_t>(rest.q.x + k.column(0)) & 15u) == 0;
    Sums x{0.0, 0.0, 0.0, 0.0};
    auto add = [&](int, double p, double q) {
        x.p += p;
        if (Against) {
            const double d = fma(-rest.c, q, p);
            x.q += q;
            x.a += if_more(d, d, p);
            x.b += if_more(q, d, p);
        }
    };
    auto all_lanes = [](double v) {
#pragma unroll
        for (uint32_t d = 16; d; d >>= 1)
            v += __shfl_xor_sync(~0u, v, d);
        return v;
    };
    uint4 wp[deep], wq[deep];
    auto load = [&](uint32_t from) { // (past the end: the last one once more)
#pragma unroll
        for (int i = 0; i < deep; ++i) {
            const int32_t at = k.column(min(from + lane + i * 32u, mine.b1 - 1u));
            wp[i] = load_block(rest.p, at, n, true);
            if (Against)
                wq[i] = load_block(rest.q, at, n, aligned);
        }
    };
    double2 upto = make_double2(0.0, 0.0);
    uint32_t part = 0, next = mine.b0 + mine.part;
    if (mine.b0 < mine.b1)
        load(mine.b0);
    for (uint32_t b = mine.b0; b < mine.b1; b += Share::kRound) {
        uint4 vp[deep], vq[deep];
#pragma unroll
        for (int i = 0; i < deep; ++i) {
            vp[i] = wp[i];
            vq[i] = Against ? wq[i] : wp[i];
        }
        load(b + Share::kRound); // on their way meanwhile
#pragma unroll
        for (int i = 0; i < deep; ++i)
            if (b + lane + i * 32u < mine.b1)
                each_weight<T, Against, Plain, Fine>(rest, k.column(b + lane + i * 32u), n, vp[i], vq[i], table, add);
        if (b + Share::kRound == next || b + Share::kRound >= mine.b1) {
            __syncwarp();
            upto = make_double2(all_lanes(Against ? x.a : x.p), Against ? all_lanes(x.b) : 0.0);
            if (lane == 0)
                s.upto[w][part] = upto;
            ++part;
            next += mine.part;
        }
    }
    if (lane >= part && lane < kParts)
        s.upto[w][lane] = upto;
    x.p = all_lanes(x.p);
    if (Against)
        x.q = all_lanes(x.q);
    x.a = upto.x;
    x.b = upto.y;
    __syncthreads(); // the sums before these have been read
    if (lane == 0)
        s.warp[w] = x;
    __syncthreads();
    Sums all{0.0, 0.0, 0.0, 0.0};
    for (uint32_t i = 0; i < kDrawWarps; ++i) {
        all.a += s.warp[i].a;
        all.b += s.warp[i].b;
        all.p += s.warp[i].p;
        all.q += s.warp[i].q;
    }
    return all;
}

// Whether all of the rows' columns count and both rows' blocks start on the same columns.
template <typename T>
__device__ __forceinline__ bool is_plain(const Rest<T>& rest)
{
    return !rest.p.mask && (!rest.against || (!rest.q.mask && ((reinterpret_cast<uintptr_t>(rest.p.x) ^ reinterpret_cast<uintptr_t>(rest.q.x)) & 15u) == 0));
}

template <typename T, bool Fine>
__device__ Sums sweep(const Rest<T>& rest, Shared& s, const Part& c)
{
    if (is_plain(rest))
        return Fine || rest.against ? sweep_rows<T, true, true, Fine>(rest, s, c) : sweep_rows<T, false, true, false>(rest, s, c);
    return Fine || rest.against ? sweep_rows<T, true, false, Fine>(rest, s, c) : sweep_rows<T, false, false, false>(rest, s, c);
}

// Of the lanes' parts x of a whole, in order: the first lane at whose end the running sum is above `want`, the last with any part
// where there is none. before: the sum in front of it. The same in every lane.
__device__ __forceinline__ uint32_t pick(double x, double want, double start, double& before)
{
    const uint32_t lane = threadIdx.x & 31u;
    double run = x;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(~0u, run, d);
        run += lane >= d ? y : 0.0;
    }
    const uint32_t some = __ballot_sync(~0u, x > kSome), reach = __ballot_sync(~0u, x > kSome && start + run > want);
    const uint32_t at = reach ? (uint32_t)__ffs(reach) - 1u : 31u - (uint32_t)__clz(some | 1u);
    before = __shfl_sync(~0u, start + (run - x), at);
    return at;
}

// The two rows' whole weights in 64 bits.
template <typename T>
__device__ double2 whole(const Row<T>& p, const Row<T>* q, Shared& s, Part& c)
{
    const double2(*all)[2] = exchange(s, c, sweep<T, false>(Rest<T>{Weigh<T>(p), Weigh<T>(q ? *q : p), q != nullptr, ~0u, 1.0}, s, c));
    double2 sum = make_double2(0.0, 0.0);
    for (uint32_t k = 0; k < c.size; ++k) {
        sum.x += all[k][1].x;
        sum.y += all[k][1].y;
    }
    return sum;
}

// The first column of the blocks [b0, b1) at which the running sum, `before` in front of them, is above `want`; the last that weighs
// anything where there is none. By the whole CTA, a block a thread.
template <typename T, bool Against, bool Fine>
__device__ __noinline__ int32_t walk(const Rest<T> rest, uint32_t b0, uint32_t b1, double before, double want, Shared& s, const Part c)
{
    constexpr int per = (int)Blocks<T>::per;
    const Blocks<T> k(rest.p.x, c.n);
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x / 32u;
    const bool aligned = (reinterpret_cast<uintptr_t>(rest.q.x + k.column(0)) & 15u) == 0;
    const uint32_t table = smem_u32(s.table);
    int32_t last = -1;
    for (uint32_t base = b0; base < b1; base += kDrawThreads) {
        double x[per], sum = 0.0;
        const uint32_t b = base + threadIdx.x;
        const int32_t i0 = k.column(min(b, b1 - 1u));
        const uint4 wp = load_block(rest.p, i0, c.n, true), wq = Against ? load_block(rest.q, i0, c.n, aligned) : wp;
        each_weight<T, Against, false, Fine>(rest, i0, c.n, wp, wq, table, [&](int e, double p, double q) {
            const double d = Against ? fma(-rest.c, q, p) : p;
            x[e] = b < b1 ? if_more(d, d, p) : 0.0; // (of P alone d is p)
        });
#pragma unroll
        for (int e = 0; e < per; ++e) {
            sum += x[e];
            last = x[e] > kSome ? i0 + e : last;
        }
        double run = sum;
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) {
            const double y = __shfl_up_sync(~0u, run, d);
            run += lane >= d ? y : 0.0;
        }
        __syncthreads();
        if (lane == 31u)
            s.run[w] = run;
        __syncthreads();
        run += before - sum;
        for (uint32_t i = 0; i < kDrawWarps; ++i) {
            run += i < w ? s.run[i] : 0.0;
            before += s.run[i];
        }
        int32_t found = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < per; ++e) {
            run += x[e];
            if (found == 0x7fffffff && x[e] > kSome && run > want)
                found = i0 + e;
        }
        if (found != 0x7fffffff)
            atomicMin(&s.token, found); // (of whole numbers: the order does not matter)
    }
    last = __reduce_max_sync(~0u, last);
    if (lane == 0)
        s.first[w] = (uint32_t)last;
    __syncthreads();
    for (uint32_t i = 0; i < kDrawWarps; ++i)
        last = max(last, (int32_t)s.first[i]);
    return s.token != 0x7fffffff ? s.token : last;
}

// The first column at which the running sum of `rest` is above u times the whole, in every CTA; -1 where the whole is nothing.
//
// The sums have the wrong sign for columns between the two c, up to |off| q of each. Rows whose p / q spread are off by the square of
// |off| over the rest, a few 1e-12; where all of Q lay between, it could be |off| over the rest. Above 1e-4 of that, which means rows
// alike to a hundredth, or where the rest is less than 1e-6 of P, the answer is kAgain: the draw is made once more, Fine, with weights
// of two terms more, whose sums are formed with the exact c (the second time off is 0: whole weights do not depend on c). From 1e-6 on
// nearly every refused draft would be drawn again: 64 sequences of four drafts 104 -> 123 us.
constexpr int32_t kAgain = -2;
template <typename T, bool Fine>
__device__ __forceinline__ int32_t draw(Rest<T> rest, double u, Shared& s, Part& c)
{
    const uint32_t lane = threadIdx.x & 31u;
    if (Fine) {
        const double2(*all)[2] = exchange(s, c, sweep<T, true>(rest, s, c));
        double2 both = make_double2(0.0, 0.0);
        for (uint32_t k = 0; k < c.size; ++k) {
            both.x += all[k][1].x;
            both.y += all[k][1].y;
        }
        rest.c = both.x / both.y;
    }
    const double2(*all)[2] = exchange(s, c, sweep<T, Fine>(rest, s, c));
    const double2 mine = lane < c.size ? all[lane][0] : make_double2(0.0, 0.0);
    double off = 0.0; // the exact c above the one that the sums were formed with
    double2 both = make_double2(0.0, 0.0);
    if (!Fine && rest.against) {
        if (lane < c.size)
            both = all[lane][1];
#pragma unroll
        for (uint32_t d = 16; d; d >>= 1) {
            both.x += __shfl_xor_sync(~0u, both.x, d);
            both.y += __shfl_xor_sync(~0u, both.y, d);
        }
        off = both.x / both.y - rest.c;
        rest.c = both.x / both.y;
    }
    const double of_cta = fma(-off, mine.y, mine.x);
    double total = of_cta, before;
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        total += __shfl_xor_sync(~0u, total, d);
    if (!Fine && rest.against && !(fabs(off) * both.y <= kLoose * total && total > kLittle * both.x))
        return kAgain;
    if (!(total > kSome))
        return -1;
    const double want = u * total;
    const uint32_t owner = pick(of_cta, want, 0.0, before);
    int32_t found = 0;
    if (c.rank == owner) { // the warp whose part holds the place
        const double of_warp = lane < kDrawWarps ? fma(-off, s.warp[lane].b, s.warp[lane].a) : 0.0;
        const uint32_t w = pick(of_warp, want, before, before);
        double2 of_part = make_double2(0.0, 0.0); // and the part of its share
        if (lane < kParts) {
            of_part = s.upto[w][lane];
            if (lane > 0)
                of_part = make_double2(of_part.x - s.upto[w][lane - 1u].x, of_part.y - s.upto[w][lane - 1u].y);
        }
        const uint32_t part = pick(fma(-off, of_part.y, of_part.x), want, before, before);
        const Share its(Blocks<T>(rest.p.x, c.n).count, c, w);
        const uint32_t b0 = its.b0 + part * its.part, b1 = min(b0 + its.part, its.b1);
        if (threadIdx.x == 0)
            s.token = 0x7fffffff;
        __syncthreads();
        found = Fine || rest.against ? walk<T, true, Fine>(rest, b0, b1, before, want, s, c) : walk<T, false, false>(rest, b0, b1, before, want, s, c);
    }
    return (int32_t)exchange(s, c, Sums{(double)found, 0.0, 0.0, 0.0})[owner][0].x;
}

// Out of the way of the others. The turn of the exchanges goes with the answer, so that no one has it in memory.
template <typename T>
__device__ __noinline__ int2 draw_fine(Rest<T> rest, double u, Shared& s, Part c)
{
    const int32_t token = draw<T, true>(rest, u, s, c);
    return make_int2(token, (int32_t)c.turn);
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 2) spec_draw_kernel(const SpecVerifyArgs a)
{
    __shared__ Shared s;
    const mk_spec_rows& r = a.r;
    const uint32_t n_drafts = r.n_pos - 1u, tid = threadIdx.x, lane = tid & 31u;
    Part c;
    c.rank = cluster_rank();
    c.size = cluster_size();
    c.n = r.n_vocab;
    c.turn = 0;
    const uint32_t sq = blockIdx.x / c.size;
    if (tid < kSteps)
        s.table[tid] = exp2((double)tid / kSteps);
    const SpecState* states = a.states + (size_t)sq * r.n_pos;
    const int32_t* drafts = r.drafts + (size_t)sq * n_drafts;
    const float* u = r.u + (size_t)sq * (r.n_pos + 1u);
    Row<T> p, q;
    heat_rows(r, sq, p, q);
    cluster_sync(); // every CTA of the cluster runs before any writes to its shared memory
    griddep_wait();
    const bool failed = __ldcg(a.failed);
    // what the first launch kept: positions up to the first that ends the round or is open
    uint32_t j = 0;
    int32_t token = -1;
    for (;;) {
        SpecState st;
        for (;;) { // a position a lane
            const uint32_t i = j + lane;
            float4 of_p = make_float4(0.0f, 0.0f, 0.0f, __uint_as_float(kEnds)), of_q = of_p;
            int32_t draft = -1;
            if (i < r.n_pos) {
                of_p = __ldcg(reinterpret_cast<const float4*>(&states[i]));
                of_q = __ldcg(reinterpret_cast<const float4*>(&states[i]) + 1);
                draft = i < n_drafts ? drafts[i] : -1;
            }
            if (failed)
                break;
            const uint32_t more = __ballot_sync(~0u, __float_as_uint(of_p.w) != kKept);
            const uint32_t kept = more ? (uint32_t)__ffs(more) - 1u : 32u;
            if (c.rank == 0 && tid < kept && (a.tokens || a.logprob)) {
                place_rows(r, sq, i, false, p, q);
                p.mass = Mass{of_p.x, of_p.y};
                if (a.tokens)
                    a.tokens[(size_t)sq * r.n_pos + i] = draft;
                if (a.logprob)
                    a.logprob[(size_t)sq * r.n_pos + i] = p.single() ? 0.0f : p.log_part(p.get((uint32_t)draft));
            }
            j += kept;
            if (!more)
                continue;
            auto from = [&](float v) { return __shfl_sync(~0u, v, kept); };
            st = SpecState{from(of_p.x), from(of_p.y), __float_as_uint(from(of_p.z)), __float_as_uint(from(of_p.w)),
                           from(of_q.x), from(of_q.y), __float_as_uint(from(of_q.z)), 0u};
            token = __shfl_sync(~0u, draft, kept);
            break;
        }
        if (failed) { // in every call from the failed one on
            if (c.rank == 0 && tid == 0) {
                a.n_kept[sq] = 0;
                a.next_token[sq] = -1;
                if (a.flags)
                    a.flags[sq] = MK_FLAG_TIMEOUT;
            }
            for (uint32_t k = tid; c.rank == 0 && k < r.n_pos; k += kDrawThreads) {
                if (a.tokens)
                    a.tokens[(size_t)sq * r.n_pos + k] = -1;
                if (a.logprob)
                    a.logprob[(size_t)sq * r.n_pos + k] = 0.0f;
            }
            return;
        }
        const int32_t d = token;
        const bool drafted = (uint32_t)d < r.n_vocab, against = drafted && r.draft_logits;
        place_rows(r, sq, j, against, p, q);
        p.weighed(Mass{st.m_p, st.s_p});
        q.weighed(Mass{st.m_q, st.s_q});
        const bool soft_q = against && !q.none() && !q.single();
        bool kept = false;
        if (p.far() || (soft_q && q.far()) || st.state == kOpen) {
            const double2 w = whole(p, soft_q ? &q : nullptr, s, c);
            p.sum64 = w.x;
            q.sum64 = w.y;
            auto part64 = [&](const Row<T>& r, uint32_t at) {
                return r.none() ? 0.0 : r.single() ? (at == (uint32_t)d ? 1.0 : 0.0) : weight_of(r, (uint32_t)d, smem_u32(s.table)) / r.sum64;
            };
            kept = drafted && (double)u[j] * (against ? part64(q, st.at_q) : 1.0) < part64(p, st.at_p);
        }
        if (kept) {
            token = d;
        } else {
            token = -1;
            const double with = (double)u[j + (drafted ? 1u : 0u)];
            if (!p.none() && p.single()) {
                token = (int32_t)st.at_p; // either the residual is there, or nothing is left and P is drawn from
            } else if (!p.none()) {
                Rest<T> rest{Weigh<T>(p), Weigh<T>(q), false, ~0u, 0.0};
                if (soft_q) {
                    rest.against = true;
                    rest.c = p.whole() / q.whole();
                } else if (against && !q.none()) {
                    rest.without = st.at_q; // all of Q: P's part there is nothing beside it
                } else if (drafted && !against) {
                    rest.without = (uint32_t)d;
                }
                for (bool all = false; token < 0 && !all;) { // where nothing is left of P, it is drawn from as a whole
                    token = draw<T, false>(rest, with, s, c);
                    if (token == kAgain) {
                        const int2 fine = draw_fine(rest, with, s, c);
                        token = fine.x;
                        c.turn = (uint32_t)fine.y;
                    }
                    all = !rest.against && rest.without == ~0u;
                    rest.against = false;
                    rest.without = ~0u;
                }
            }
        }
        if (c.rank == 0 && tid == 0) {
            if (a.tokens)
                a.tokens[(size_t)sq * r.n_pos + j] = token;
            if (a.logprob)
                a.logprob[(size_t)sq * r.n_pos + j] = token < 0 || p.single() ? 0.0f : p.log_part(p.get((uint32_t)token));
        }
        if (!kept)
            break;
        ++j;
    }
    if (c.rank == 0) {
        if (tid == 0) {
            a.n_kept[sq] = (int32_t)j;
            a.next_token[sq] = token;
            a.ended[sq] = 0; // the next call finds its counters as this one did
            if (sq == 0)
                *a.counter = 0;
        }
        for (uint32_t k = tid; k < r.n_pos; k += kDrawThreads)
            a.tickets[(size_t)sq * r.n_pos + k] = 0;
        uint32_t flags = 0;
        if (token < 0) {
            uint32_t any = p.mask == nullptr;
            for (uint32_t i = tid; p.mask && i < (r.n_vocab + 31u) / 32u; i += kDrawThreads)
                any |= p.mask[i] & (r.n_vocab - i * 32u < 32u ? (1u << (r.n_vocab - i * 32u)) - 1u : ~0u);
            flags = MK_FLAG_NO_CANDIDATE | (__syncthreads_or(any != 0) ? 0u : MK_FLAG_ALL_MASKED);
        }
        if (tid == 0 && a.flags)
            a.flags[sq] = flags;
        for (uint32_t k = j + 1u + tid; k < r.n_pos; k += kDrawThreads) {
            if (a.tokens)
                a.tokens[(size_t)sq * r.n_pos + k] = -1;
            if (a.logprob)
                a.logprob[(size_t)sq * r.n_pos + k] = 0.0f;
        }
    }
    cluster_sync(); // nothing is sent to a CTA that has gone
}

// How many of the draw's clusters of a size fit on the device: fewer than its CTAs would make, as a cluster lies within a part of the
// chip (of 296 CTAs 14 clusters of 16, 33 of 8, 71 of 4). Asked for once on each of the first 64 devices.
template <typename T>
cudaError_t resident_clusters(uint32_t size, uint32_t& fit)
{
    static std::atomic<int> known[64][kMaxCluster + 1];
    static std::atomic<uint64_t> wide_set{0};
    int device = 0, n = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && size > 8)
        e = set_once(wide_set, spec_draw_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess)
        return e;
    if (device < 64 && (n = known[device][size].load(std::memory_order_relaxed)) != 0) {
        fit = (uint32_t)n - 1u;
        return e;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(size);
    c.blockDim = dim3(kDrawThreads);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    c.attrs = attr;
    c.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, spec_draw_kernel<T>, &c);
    if (e != cudaSuccess)
        return e;
    fit = n > 0 ? (uint32_t)n : 0u;
    if (device < 64)
        known[device][size].store((int)fit + 1, std::memory_order_relaxed);
    return e;
}

template <typename T>
cudaError_t launch(SpecVerifyArgs a, cudaStream_t stream)
{
    const uint32_t n = a.r.n_seq, rows = n * a.r.n_pos;
    // Slices of about 64 KB a row; smaller ones where that leaves CTAs without work, down to 4 KB.
    const uint32_t bytes = a.r.n_vocab * (uint32_t)sizeof(T), room = (2u * kScanCtas + rows - 1) / rows, most = (bytes + 4095u) / 4096u;
    uint32_t slices = (bytes + 65535u) / 65536u;
    slices = slices > room ? slices : room;
    slices = slices < a.slices ? slices : a.slices;
    a.slices = slices < most ? slices : most;
    static std::atomic<uint64_t> scan_set{0};
    cudaError_t e = set_once(scan_set, spec_scan_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kTiles * kTileBytes));
    if (e != cudaSuccess)
        return e;
    // The largest clusters of which all are resident at once: a second wave takes as long as the first (18 sequences of 129280 columns
    // by 16 CTAs 49 us, by 8 37; 37 by 8 54, by 4 43; 74 by 4 65, by 2 57; 148 by 2 70, by one 91; 149 by 2 97, by one 90).
    uint32_t size = kMaxCluster;
    while (size > 1 && a.r.n_vocab < size * 1024u)
        size >>= 1;
    for (; size > 1; size >>= 1) {
        uint32_t fit = 0;
        e = resident_clusters<T>(size, fit);
        if (e != cudaSuccess)
            return e;
        if (n <= fit)
            break;
    }
    const uint32_t work = rows * a.slices;
    spec_scan_kernel<T><<<work < kScanCtas ? work : kScanCtas, kScanThreads, kTiles * kTileBytes, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(n * size);
    c.blockDim = dim3(kDrawThreads);
    c.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = 2;
    return cudaLaunchKernelEx(&c, spec_draw_kernel<T>, a);
}

} // namespace

cudaError_t launch_spec_verify(const SpecVerifyArgs& a, cudaStream_t stream)
{
    switch (a.r.type) {
    case MK_FP32: return launch<float>(a, stream);
    case MK_BF16: return launch<__nv_bfloat16>(a, stream);
    default: return launch<__half>(a, stream);
    }
}

} // namespace mk
