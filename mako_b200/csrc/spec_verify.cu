// Verification of a speculative round against whole distributions (mk_spec_verify in include/mako_b200.h). A cluster of CTAs per
// sequence, each with a slice of the vocabulary, walks the sequence's positions and stops where the round ends: the rows behind
// the first refused draft, about half of them as drafters go, are never read. What bounds it is the reading of the rows up to
// there; the clusters of a launch are at different places of their sequences, so that one's decisions run beside another's reads.
//
// A position: one pass over the target's row and the drafter's, each thread with its own running maximum and sum of
// exp2((x - max) log2(e) / T), fp32; the slices' maxima and sums meet through distributed shared memory (one cluster barrier), and
// every CTA comes to the same decision. These sums are good to about 1e-6; a decision nearer than kNear is taken again with the
// sums of the draw.
//
// The draw, once a sequence: in a vocabulary's running sum every token lies next to others, so weights and sums are in 64 bits
// here, from rows that are in L2 by then: exp2 by a table of 1024 steps and a quadratic (error 1e-11, of either sign). Where a
// drafter's row takes part, a pass for the two sums and one for max(0, P - Q); else a single one. The sums by CTA and warp lead to
// one warp's columns, which the CTA goes over once more, eight columns a thread.
#include "ptx.cuh"
#include "round_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

constexpr uint32_t kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32, kMaxCluster = 16;
constexpr uint32_t kSteps = 1024; // of the table of exp2
constexpr float kNear = 3e-5f;    // decisions nearer than this, relative, are taken in 64 bits
constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

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

// A maximum and the sum of weights relative to it; -inf and 0 where there is none.
struct Mass {
    float m, s;
    __device__ void add(const Mass& o, float scale)
    {
        const float top = fmaxf(m, o.m);
        if (top == -kInf || top == kInf) { // nothing yet, or a sum that no one will use
            m = top;
            return;
        }
        s = s * ex2_approx((m - top) * scale) + o.s * ex2_approx((o.m - top) * scale);
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
    Mass mass;            // of the whole row
    __device__ void temperature(float v)
    {
        t = v > 0.0f && v < kInf ? v : 0.0f;
        scale64 = t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
        scale = (float)fmin(scale64, 3e38);
    }
    __device__ bool none() const { return mass.m == -kInf; }
    __device__ bool single() const { return t == 0.0f || mass.m == kInf; }
    // A column's logit; what is masked or NaN is -inf.
    __device__ float get(uint32_t i) const
    {
        const bool off = mask && !((__ldg(mask + (i >> 5)) >> (i & 31u)) & 1u);
        return off ? -kInf : fmaxf(to_float(x[i]), -kInf);
    }
};

struct Shared {
    double table[kSteps];
    double2 slices[2][kMaxCluster]; // what each CTA of the cluster sent, in turns
    double warp_p[kVerifyWarps], warp_q[kVerifyWarps];
    Mass mass_p[kVerifyWarps], mass_q[kVerifyWarps];
    uint32_t first[kVerifyWarps];
    int32_t token;
};

// One CTA's part in a cluster: its slice of the columns, and the turn of the exchanges.
struct Part {
    uint32_t rank, size, n, from, to, turn;
};

// Sends (a, b), the same in the first `size` threads, to every CTA; after it slices[turn] has all.
__device__ __forceinline__ const double2* exchange(Shared& s, Part& c, double a, double b)
{
    const double2* got = s.slices[c.turn];
    if (threadIdx.x < c.size)
        put(in_cta(&s.slices[c.turn][c.rank], threadIdx.x), a, b);
    c.turn ^= 1u;
    cluster_sync();
    return got;
}

// A thread's share of the row's columns [from, to): 16 bytes at a time where they are whole, kDeep of them under way.
template <typename T>
__device__ __forceinline__ Mass scan(const Row<T>& r, const Part& c)
{
    constexpr uint32_t per = 16 / sizeof(T);
    constexpr int kDeep = 4;
    Mass a{-kInf, 0.0f};
    auto one = [&](uint32_t i) { a.add(Mass{r.get(i), 1.0f}, r.scale); };
    // columns in front of the slice's first 16-byte boundary, and behind its last
    const uint32_t odd = (uint32_t)((reinterpret_cast<uintptr_t>(r.x + c.from) & 15u) / sizeof(T));
    const uint32_t head = min(odd ? per - odd : 0u, c.to - c.from);
    const uint32_t first = c.from + head, blocks = (c.to - first) / per;
    if (threadIdx.x < head)
        one(c.from + threadIdx.x);
    const uint32_t behind = first + blocks * per + threadIdx.x;
    if (behind < c.to)
        one(behind);
    const uint4* x = reinterpret_cast<const uint4*>(r.x + first);
    for (uint32_t b = threadIdx.x; b < blocks; b += kDeep * kVerifyThreads) {
        uint4 w[kDeep];
        uint32_t on[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const uint32_t at = b + k * kVerifyThreads;
            on[k] = at < blocks ? (1u << per) - 1u : 0u;
            if (r.mask && at < blocks) {
                const uint32_t i = first + at * per, lo = __ldg(r.mask + (i >> 5)), hi = __ldg(r.mask + ((i + per - 1u) >> 5));
                on[k] &= __funnelshift_r(lo, hi, i & 31u);
            }
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
            w[k] = on[k] ? __ldg(x + b + k * kVerifyThreads) : make_uint4(0, 0, 0, 0);
        float v[kDeep][per], top = -kInf;
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
#pragma unroll
            for (int e = 0; e < (int)per; ++e) {
                const T y = reinterpret_cast<const T*>(&w[k])[e];
                v[k][e] = on[k] >> e & 1u ? fmaxf(to_float(y), -kInf) : -kInf;
                top = fmaxf(top, v[k][e]);
            }
        if (top > a.m) {
            a.s = a.m == -kInf ? 0.0f : a.s * ex2_approx((a.m - top) * r.scale);
            a.m = top;
        }
        if (a.m > -kInf && a.m < kInf) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kDeep; ++k)
#pragma unroll
                for (int e = 0; e < (int)per; ++e)
                    sum += ex2_approx((v[k][e] - a.m) * r.scale);
            a.s += sum;
        }
    }
    return a;
}

__device__ __forceinline__ Mass warp_mass(Mass a, float scale)
{
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        const Mass o{__shfl_xor_sync(~0u, a.m, d), __shfl_xor_sync(~0u, a.s, d)};
        // the lower lane's first in both, so that the two come to the same bits
        Mass x = threadIdx.x & d ? o : a;
        x.add(threadIdx.x & d ? a : o, scale);
        a = x;
    }
    return a;
}

// The two rows' masses (q: or none), the same in every thread of the cluster.
template <typename T>
__device__ void weigh(Row<T>& p, Row<T>* q, Shared& s, Part& c)
{
    const Mass a = warp_mass(scan(p, c), p.scale);
    const Mass b = q ? warp_mass(scan(*q, c), q->scale) : Mass{-kInf, 0.0f};
    if ((threadIdx.x & 31u) == 0) {
        s.mass_p[threadIdx.x / 32u] = a;
        s.mass_q[threadIdx.x / 32u] = b;
    }
    __syncthreads();
    Mass x = s.mass_p[0], y = s.mass_q[0];
    if (threadIdx.x < 32) {
        for (uint32_t w = 1; w < kVerifyWarps; ++w) {
            x.add(s.mass_p[w], p.scale);
            if (q)
                y.add(s.mass_q[w], q->scale);
        }
    }
    const double2* all = exchange(s, c, __hiloint2double(__float_as_int(x.m), __float_as_int(x.s)),
                                  __hiloint2double(__float_as_int(y.m), __float_as_int(y.s)));
    auto open = [](double d) { return Mass{__int_as_float(__double2hiint(d)), __int_as_float(__double2loint(d))}; };
    p.mass = open(all[0].x);
    for (uint32_t r = 1; r < c.size; ++r)
        p.mass.add(open(all[r].x), p.scale);
    if (q) {
        q->mass = open(all[0].y);
        for (uint32_t r = 1; r < c.size; ++r)
            q->mass.add(open(all[r].y), q->scale);
    }
}

// The first column of the row that holds its largest logit.
template <typename T>
__device__ uint32_t first_of_largest(const Row<T>& r, Shared& s, Part& c)
{
    uint32_t at = ~0u;
    for (uint32_t i = c.from + threadIdx.x; i < c.to && at == ~0u; i += kVerifyThreads)
        if (r.get(i) == r.mass.m)
            at = i;
    at = __reduce_min_sync(~0u, at);
    if ((threadIdx.x & 31u) == 0)
        s.first[threadIdx.x / 32u] = at;
    __syncthreads();
    for (uint32_t w = 0; w < kVerifyWarps; ++w)
        at = min(at, s.first[w]);
    const double2* all = exchange(s, c, (double)at, 0.0);
    double best = all[0].x;
    for (uint32_t k = 1; k < c.size; ++k)
        best = fmin(best, all[k].x);
    return (uint32_t)best;
}

// 2^((x - m) scale) in 64 bits, x <= m: 2^(k/1024) from the table times a quadratic of the rest, |r| <= 1/2048 of a power:
// (r ln2)^3 / 6 = 6.5e-12 at most.
__device__ __forceinline__ double weight64(float x, float m, double scale, const double* table)
{
    const double t = ((double)x - (double)m) * (scale * kSteps);
    if (!(t > -1000.0 * kSteps)) // 2^-1000: nothing, even to the sum of a vocabulary; and -inf
        return 0.0;
    const double shift = 6755399441055744.0; // 1.5 * 2^52: the sum's low bits are t to the nearest whole
    const double k = t + shift;
    const long long n = __double_as_longlong(k); // low bits: the whole part
    const double r = (t - (k - shift)) * (0.6931471805599453 / kSteps);
    const double y = table[n & (long long)(kSteps - 1)];
    const double z = fma(y, fma(0.5 * r, r, r), y);
    const int e = (int)(uint32_t)n >> 10; // arithmetic: the power of two
    return __hiloint2double(__double2hiint(z) + e * (1 << 20), __double2loint(z));
}

template <typename T>
__device__ __forceinline__ double weight64(const Row<T>& r, uint32_t i, const double* table)
{
    return weight64(r.get(i), r.mass.m, r.scale64, table);
}

// What a draw draws from: of column i max(0, P - Q), not normalised where Q is one draft alone or none.
template <typename T>
struct Rest {
    const Row<T>*p, *q;
    uint32_t without;       // column that weighs nothing, or ~0
    double inv_p, inv_q;
    __device__ double at(uint32_t i, const double* table) const
    {
        const double w = weight64(*p, i, table);
        if (!q)
            return i == without ? 0.0 : w;
        return fmax(w * inv_p - weight64(*q, i, table) * inv_q, 0.0);
    }
};

// Columns of a warp's part in a sweep: a slice is dealt out to the warps in order.
__device__ __forceinline__ uint32_t warp_part(const Part& c) { return (c.to - c.from + kVerifyWarps - 1) / kVerifyWarps; }

// Sums of f(i) and g(i) over the CTA's slice, by warp, left in s.warp_p and s.warp_q and returned for the CTA.
template <typename F>
__device__ __forceinline__ double2 sweep(Shared& s, const Part& c, F f)
{
    const uint32_t w = threadIdx.x / 32u, per = warp_part(c);
    const uint32_t from = min(c.from + w * per, c.to), to = min(from + per, c.to);
    double a = 0.0, b = 0.0;
#pragma unroll 4
    for (uint32_t i = from + (threadIdx.x & 31u); i < to; i += 32) {
        const double2 x = f(i);
        a += x.x;
        b += x.y;
    }
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        a += __shfl_xor_sync(~0u, a, d);
        b += __shfl_xor_sync(~0u, b, d);
    }
    __syncthreads(); // the sums before these have been read
    if ((threadIdx.x & 31u) == 0) {
        s.warp_p[w] = a;
        s.warp_q[w] = b;
    }
    __syncthreads();
    double2 all = make_double2(0.0, 0.0);
    for (uint32_t i = 0; i < kVerifyWarps; ++i) {
        all.x += s.warp_p[i];
        all.y += s.warp_q[i];
    }
    return all;
}

// The two rows' whole weights in 64 bits.
template <typename T>
__device__ double2 whole(const Row<T>& p, const Row<T>* q, Shared& s, Part& c)
{
    const double2 mine = sweep(s, c, [&](uint32_t i) {
        return make_double2(weight64(p, i, s.table), q ? weight64(*q, i, s.table) : 0.0);
    });
    const double2* all = exchange(s, c, mine.x, mine.y);
    double2 sum = make_double2(0.0, 0.0);
    for (uint32_t k = 0; k < c.size; ++k) {
        sum.x += all[k].x;
        sum.y += all[k].y;
    }
    return sum;
}

// The first column at which the running sum of `rest` is above u times the whole, in every CTA; -1 where the whole is nothing.
template <typename T>
__device__ int32_t draw(const Rest<T>& rest, double u, Shared& s, Part& c)
{
    const double mine = sweep(s, c, [&](uint32_t i) { return make_double2(rest.at(i, s.table), 0.0); }).x;
    const double2* all = exchange(s, c, mine, 0.0);
    double total = 0.0;
    for (uint32_t k = 0; k < c.size; ++k)
        total += all[k].x;
    if (!(total > 0.0))
        return -1;
    // the CTA, then the warp whose columns hold the place; the last with any where rounding leaves none
    const double want = u * total;
    double before = 0.0, at_before = 0.0;
    uint32_t owner = 0;
    for (uint32_t k = 0; k < c.size; ++k) {
        if (all[k].x > 0.0) {
            owner = k;
            at_before = before;
            if (before + all[k].x > want)
                break;
        }
        before += all[k].x;
    }
    if (c.rank == owner) {
        before = at_before;
        uint32_t w = 0;
        for (uint32_t k = 0; k < kVerifyWarps; ++k) {
            if (s.warp_p[k] > 0.0) {
                w = k;
                at_before = before;
                if (before + s.warp_p[k] > want)
                    break;
            }
            before += s.warp_p[k];
        }
        before = at_before;
        const uint32_t per = warp_part(c), from = min(c.from + w * per, c.to), to = min(from + per, c.to);
        int32_t last = -1;
        __syncthreads(); // warp_p is used again below
        if (threadIdx.x == 0)
            s.token = 0x7fffffff;
        // eight columns a thread, in order
        constexpr uint32_t kEach = 8;
        for (uint32_t base = from; base < to; base += kEach * kVerifyThreads) {
            double x[kEach], sum = 0.0;
            const uint32_t i0 = base + threadIdx.x * kEach;
#pragma unroll
            for (uint32_t k = 0; k < kEach; ++k) {
                x[k] = i0 + k < to ? rest.at(i0 + k, s.table) : 0.0;
                sum += x[k];
                last = x[k] > 0.0 ? (int32_t)(i0 + k) : last;
            }
            double run = sum;
#pragma unroll
            for (uint32_t d = 1; d < 32; d <<= 1) {
                const double y = __shfl_up_sync(~0u, run, d);
                run += (threadIdx.x & 31u) >= d ? y : 0.0;
            }
            __syncthreads();
            if ((threadIdx.x & 31u) == 31u)
                s.warp_p[threadIdx.x / 32u] = run;
            __syncthreads();
            run += before - sum;
            for (uint32_t k = 0; k < kVerifyWarps; ++k) {
                run += k < threadIdx.x / 32u ? s.warp_p[k] : 0.0;
                before += s.warp_p[k];
            }
            int32_t found = 0x7fffffff;
#pragma unroll
            for (uint32_t k = 0; k < kEach; ++k) {
                run += x[k];
                if (found == 0x7fffffff && x[k] > 0.0 && run > want)
                    found = (int32_t)(i0 + k);
            }
            if (found != 0x7fffffff)
                atomicMin(&s.token, found); // (of whole numbers: the order does not matter)
        }
        last = __reduce_max_sync(~0u, last);
        if ((threadIdx.x & 31u) == 0)
            s.first[threadIdx.x / 32u] = (uint32_t)last;
        __syncthreads();
        for (uint32_t k = 0; k < kVerifyWarps; ++k)
            last = max(last, (int32_t)s.first[k]);
        const int32_t found = s.token != 0x7fffffff ? s.token : last;
        exchange(s, c, (double)found, 0.0);
        return found;
    }
    return (int32_t)exchange(s, c, 0.0, 0.0)[owner].x;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 3) spec_verify_kernel(const SpecVerifyArgs a)
{
    __shared__ Shared s;
    const mk_spec_rows& r = a.r;
    const uint32_t n_drafts = r.n_pos - 1u, tid = threadIdx.x;
    Part c;
    c.rank = cluster_rank();
    c.size = cluster_size();
    c.n = r.n_vocab;
    const uint32_t per = (((c.n + c.size - 1) / c.size) + 31u) & ~31u;
    c.from = min(c.rank * per, c.n);
    c.to = min(c.from + per, c.n);
    c.turn = 0;
    const uint32_t sq = blockIdx.x / c.size;
    for (uint32_t i = tid; i < kSteps; i += kVerifyThreads)
        s.table[i] = exp2((double)i / kSteps);
    Row<T> p, q;
    p.temperature(r.temperature ? r.temperature[sq] : r.temperature_all);
    q.temperature(r.draft_temperature ? r.draft_temperature[sq] : r.temperature ? r.temperature[sq] : r.temperature_all);
    const float* u = r.u + (size_t)sq * (r.n_pos + 1u);
    const bool writes = c.rank == 0 && tid == 0;
    cluster_sync(); // every CTA of the cluster runs before any writes to its shared memory
    uint32_t j = 0;
    int32_t token = -1;
    for (;; ++j) {
        const size_t row = (size_t)sq * r.n_pos + j, drow = (size_t)sq * n_drafts + j;
        const int32_t d = j < n_drafts ? r.drafts[drow] : -1;
        const bool drafted = d >= 0 && (uint32_t)d < r.n_vocab, against = drafted && r.draft_logits;
        p.x = static_cast<const T*>(r.logits) + row * r.ld;
        p.mask = r.mask ? r.mask + row * r.mask_ld : nullptr;
        q.x = against ? static_cast<const T*>(r.draft_logits) + drow * r.draft_ld : nullptr;
        q.mask = r.mask_drafts ? p.mask : nullptr;
        const float x = drafted ? p.get((uint32_t)d) : 0.0f, y = against ? q.get((uint32_t)d) : 0.0f, uj = u[j];
        weigh(p, against ? &q : nullptr, s, c);
        // where a row's weight is all on one place
        uint32_t at_p = ~0u, at_q = ~0u;
        if (!p.none() && p.single())
            at_p = first_of_largest(p, s, c);
        if (against && !q.none() && q.single())
            at_q = first_of_largest(q, s, c);
        auto part = [](const Row<T>& r, float x, uint32_t at, uint32_t d) {
            return r.none() ? 0.0f : r.single() ? (at == d ? 1.0f : 0.0f) : ex2_approx((x - r.mass.m) * r.scale) / r.mass.s;
        };
        bool kept = false;
        double2 w = make_double2(0.0, 0.0);
        if (drafted) {
            const float pd = part(p, x, at_p, (uint32_t)d), qd = against ? part(q, y, at_q, (uint32_t)d) : 1.0f;
            const float lhs = uj * qd;
            kept = lhs < pd;
            const bool soft = !p.none() && (!p.single() || (against && !q.none() && !q.single()));
            if (soft && fabsf(lhs - pd) <= kNear * fmaxf(lhs, pd)) {
                w = whole(p, against ? &q : nullptr, s, c);
                auto part64 = [&](const Row<T>& r, float x, uint32_t at, double all) {
                    return r.none() ? 0.0 : r.single() ? (at == (uint32_t)d ? 1.0 : 0.0) : weight64(x, r.mass.m, r.scale64, s.table) / all;
                };
                kept = (double)uj * (against ? part64(q, y, at_q, w.y) : 1.0) < part64(p, x, at_p, w.x);
            }
        }
        if (kept) {
            token = d;
        } else {
            token = -1;
            const double with = (double)(drafted ? u[j + 1] : uj);
            if (p.none()) {
            } else if (p.single()) {
                token = (int32_t)at_p; // either the residual is there, or nothing is left and P is drawn from
            } else {
                if (against && !q.none()) {
                    if (q.single()) {
                        // P without what Q takes of one place, where Q has all: that place is left with nothing
                        token = draw(Rest<T>{&p, nullptr, at_q, 0.0, 0.0}, with, s, c);
                    } else {
                        w = whole(p, &q, s, c);
                        token = draw(Rest<T>{&p, &q, ~0u, 1.0 / w.x, 1.0 / w.y}, with, s, c);
                    }
                } else if (drafted && !against) {
                    token = draw(Rest<T>{&p, nullptr, (uint32_t)d, 0.0, 0.0}, with, s, c);
                }
                if (token < 0)
                    token = draw(Rest<T>{&p, nullptr, ~0u, 0.0, 0.0}, with, s, c);
            }
        }
        if (writes) {
            if (a.tokens)
                a.tokens[row] = token;
            if (a.logprob)
                a.logprob[row] = token < 0 || p.single() ? 0.0f
                                                         : (float)(((double)p.get((uint32_t)token) - (double)p.mass.m) / (double)p.t) - logf(p.mass.s);
        }
        if (!kept)
            break;
    }
    if (writes) {
        a.n_kept[sq] = (int32_t)j;
        a.next_token[sq] = token;
    }
    if (c.rank == 0) {
        uint32_t flags = 0;
        if (token < 0) {
            uint32_t any = p.mask == nullptr;
            for (uint32_t i = tid; p.mask && i < (r.n_vocab + 31u) / 32u; i += kVerifyThreads)
                any |= p.mask[i] & (r.n_vocab - i * 32u < 32u ? (1u << (r.n_vocab - i * 32u)) - 1u : ~0u);
            flags = MK_FLAG_NO_CANDIDATE | (__syncthreads_or(any != 0) ? 0u : MK_FLAG_ALL_MASKED);
        }
        if (tid == 0 && a.flags)
            a.flags[sq] = flags;
        for (uint32_t k = j + 1u + tid; k < r.n_pos; k += kVerifyThreads) {
            if (a.tokens)
                a.tokens[(size_t)sq * r.n_pos + k] = -1;
            if (a.logprob)
                a.logprob[(size_t)sq * r.n_pos + k] = 0.0f;
        }
    }
    cluster_sync(); // nothing is sent to a CTA that has gone
}

template <typename T>
cudaError_t launch(const SpecVerifyArgs& a, cudaStream_t stream)
{
    // As many CTAs as are resident at once, three or four on each SM, in clusters of up to eight (sixteen for a few sequences).
    const uint32_t n = a.r.n_seq;
    uint32_t size = n <= 8 ? 16u : n <= 72 ? 8u : n <= 144 ? 4u : 2u;
    while (size > 1 && a.r.n_vocab < size * 1024u)
        size >>= 1;
    if (size > 8) {
        const cudaError_t e = cudaFuncSetAttribute(spec_verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess)
            return e;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(n * size);
    c.blockDim = dim3(kVerifyThreads);
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    c.attrs = attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, spec_verify_kernel<T>, a);
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
