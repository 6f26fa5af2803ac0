// Verification of a speculative round against whole distributions (mk_spec_verify in include/mako_b200.h). One CTA per sequence
// walks its positions and stops where the round ends, so that the rows behind it are never read.
#include "ptx.cuh"
#include "round_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

constexpr uint32_t kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
struct Row {
    const T* x;
    const uint32_t* mask; // or nullptr
    uint32_t n;
    double inv_t; // 0: all weight on one place
    // what stats() finds
    unsigned long long best; // (order key of the largest, ~its place); key 0: all NaN
    float m;
    bool none, single; // nothing weighs anything; all weight on one place
    uint32_t at;
    double sum;
    __device__ float get(uint32_t i) const
    {
        const bool off = mask && !((mask[i >> 5] >> (i & 31u)) & 1u);
        return off ? __int_as_float(0xff800000) : to_float(x[i]);
    }
    // Weight of column i relative to the largest.
    __device__ double weight(uint32_t i) const
    {
        if (none)
            return 0.0;
        if (single)
            return i == at ? 1.0 : 0.0;
        const float v = get(i);
        return v > __int_as_float(0xff800000) ? exp(((double)v - (double)m) * inv_t) : 0.0;
    }
    __device__ double p(uint32_t i) const { return none ? 0.0 : weight(i) / sum; }
};

struct Shared {
    unsigned long long key[kVerifyWarps];
    double part[kVerifyWarps];
    int32_t token;
    int32_t last[kVerifyWarps];
};

__device__ unsigned long long block_max(Shared& s, unsigned long long k)
{
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        const unsigned long long o = __shfl_xor_sync(~0u, k, d);
        k = o > k ? o : k;
    }
    __syncthreads();
    if ((threadIdx.x & 31u) == 0)
        s.key[threadIdx.x >> 5] = k;
    __syncthreads();
    for (uint32_t w = 0; w < kVerifyWarps; ++w)
        k = s.key[w] > k ? s.key[w] : k;
    return k;
}

__device__ double block_sum(Shared& s, double x)
{
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        x += __shfl_xor_sync(~0u, x, d);
    __syncthreads();
    if ((threadIdx.x & 31u) == 0)
        s.part[threadIdx.x >> 5] = x;
    __syncthreads();
    double all = 0.0;
    for (uint32_t w = 0; w < kVerifyWarps; ++w)
        all += s.part[w];
    return all;
}

template <typename T>
__device__ void stats(Row<T>& r, Shared& s)
{
    unsigned long long k = 0;
    for (uint32_t i = threadIdx.x; i < r.n; i += kVerifyThreads) {
        const unsigned long long o = ((unsigned long long)order_key(r.get(i)) << 32) | (uint32_t)~i;
        k = o > k ? o : k;
    }
    k = block_max(s, k);
    r.m = key_to_float((uint32_t)(k >> 32));
    r.at = ~(uint32_t)k;
    r.none = (k >> 32) == 0 || r.m == __int_as_float(0xff800000);
    r.single = r.inv_t == 0.0 || r.m == __int_as_float(0x7f800000);
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < r.n; i += kVerifyThreads)
        sum += r.weight(i);
    r.sum = block_sum(s, sum);
}

__device__ double inverse(float t) { return t > 0.0f ? 1.0 / (double)t : 0.0; }

// The first column at which the running sum of max(0, P - Q) is above u times the whole; -1 where the whole is nothing.
// q: nullptr: all of Q on `certain` (none where that is negative).
template <typename T>
__device__ int32_t draw(const Row<T>& p, const Row<T>* q, int32_t certain, double u, Shared& s)
{
    auto rest = [&](uint32_t i) {
        const double x = p.p(i) - (q ? q->p(i) : (int32_t)i == certain ? 1.0 : 0.0);
        return x > 0.0 ? x : 0.0;
    };
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
    const uint32_t per = (p.n + kVerifyWarps - 1) / kVerifyWarps;
    const uint32_t from = min(w * per, p.n), to = min(from + per, p.n);
    double sum = 0.0;
    int32_t last = -1;
    for (uint32_t i = from + lane; i < to; i += 32) {
        const double x = rest(i);
        sum += x;
        last = x > 0.0 ? (int32_t)i : last;
    }
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, d);
        last = max(last, __shfl_xor_sync(~0u, last, d));
    }
    __syncthreads();
    if (lane == 0) {
        s.part[w] = sum;
        s.last[w] = last;
    }
    __syncthreads();
    double all = 0.0;
    int32_t end = -1, mine = -1;
    for (uint32_t i = 0; i < kVerifyWarps; ++i)
        all += s.part[i];
    const double want = u * all;
    double before = 0.0;
    for (uint32_t i = 0; i < kVerifyWarps; ++i) {
        if (s.last[i] >= 0) {
            end = (int32_t)i;
            if (mine < 0 && before + s.part[i] > want)
                mine = (int32_t)i;
        }
        before += mine < 0 ? s.part[i] : 0.0;
    }
    if (end < 0)
        return -1;
    if (mine < 0) { // u times the whole rounds to the whole: the last of all
        mine = end;
        before = 0.0;
        for (int32_t i = 0; i < mine; ++i)
            before += s.part[i];
    }
    if ((int32_t)w == mine) {
        int32_t found = s.last[w];
        for (uint32_t base = from; base < to; base += 32) {
            const uint32_t i = base + lane;
            const double x = i < to ? rest(i) : 0.0;
            double run = x;
#pragma unroll
            for (uint32_t d = 1; d < 32; d <<= 1) {
                const double y = __shfl_up_sync(~0u, run, d);
                run += lane >= d ? y : 0.0;
            }
            const uint32_t hit = __ballot_sync(~0u, x > 0.0 && before + run > want);
            if (hit) {
                found = (int32_t)(base + __ffs(hit) - 1);
                break;
            }
            before += __shfl_sync(~0u, run, 31);
        }
        if (lane == 0)
            s.token = found;
    }
    __syncthreads();
    return s.token;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) spec_verify_kernel(const SpecVerifyArgs a)
{
    __shared__ Shared s;
    const mk_spec_rows& r = a.r;
    const uint32_t sq = blockIdx.x, n_drafts = r.n_pos - 1u, tid = threadIdx.x;
    const float t = r.temperature ? r.temperature[sq] : r.temperature_all;
    Row<T> p, q;
    p.n = q.n = r.n_vocab;
    p.inv_t = inverse(t);
    q.inv_t = inverse(r.draft_temperature ? r.draft_temperature[sq] : t);
    const float* u = r.u + (size_t)sq * (r.n_pos + 1u);
    uint32_t j = 0;
    int32_t token = -1;
    for (;; ++j) {
        const size_t row = (size_t)sq * r.n_pos + j, drow = (size_t)sq * n_drafts + j;
        const int32_t d = j < n_drafts ? r.drafts[drow] : -1;
        const bool drafted = d >= 0 && (uint32_t)d < r.n_vocab;
        p.x = static_cast<const T*>(r.logits) + row * r.ld;
        p.mask = r.mask ? r.mask + row * r.mask_ld : nullptr;
        stats(p, s);
        double qd = 1.0;
        if (drafted && r.draft_logits) {
            q.x = static_cast<const T*>(r.draft_logits) + drow * r.draft_ld;
            q.mask = r.mask_drafts ? p.mask : nullptr;
            stats(q, s);
            qd = q.p((uint32_t)d);
        }
        if (drafted && (double)u[j] * qd < p.p((uint32_t)d)) {
            token = d;
        } else {
            token = -1;
            if (drafted)
                token = draw(p, r.draft_logits ? &q : nullptr, d, (double)u[j + 1], s);
            if (token < 0)
                token = draw<T>(p, nullptr, -1, (double)u[j + (drafted ? 1 : 0)], s);
        }
        if (tid == 0) {
            if (a.tokens)
                a.tokens[row] = token;
            if (a.logprob)
                a.logprob[row] = token < 0 ? 0.0f : (float)log(p.p((uint32_t)token));
        }
        if (!drafted || token != d || !((double)u[j] * qd < p.p((uint32_t)d)))
            break;
    }
    if (tid == 0) {
        a.n_kept[sq] = (int32_t)j;
        a.next_token[sq] = token;
        if (a.flags)
            a.flags[sq] = token < 0 ? MK_FLAG_NO_CANDIDATE : 0u;
    }
    if (token < 0 && a.flags && p.mask) {
        uint32_t any = 0;
        for (uint32_t i = tid; i < (r.n_vocab + 31u) / 32u; i += kVerifyThreads)
            any |= p.mask[i] & (r.n_vocab - i * 32u < 32u ? (1u << (r.n_vocab - i * 32u)) - 1u : ~0u);
        if (!__syncthreads_or(any != 0) && tid == 0)
            a.flags[sq] |= MK_FLAG_ALL_MASKED;
    }
    for (uint32_t k = j + 1u + tid; k < r.n_pos; k += kVerifyThreads) {
        if (a.tokens)
            a.tokens[(size_t)sq * r.n_pos + k] = -1;
        if (a.logprob)
            a.logprob[(size_t)sq * r.n_pos + k] = 0.0f;
    }
}

} // namespace

cudaError_t launch_spec_verify(const SpecVerifyArgs& a, cudaStream_t stream)
{
    switch (a.r.type) {
    case MK_FP32: spec_verify_kernel<float><<<a.r.n_seq, kVerifyThreads, 0, stream>>>(a); break;
    case MK_BF16: spec_verify_kernel<__nv_bfloat16><<<a.r.n_seq, kVerifyThreads, 0, stream>>>(a); break;
    default: spec_verify_kernel<__half><<<a.r.n_seq, kVerifyThreads, 0, stream>>>(a); break;
    }
    return cudaGetLastError();
}

} // namespace mk
