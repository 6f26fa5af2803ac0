// Rotated keys and values into a paged cache of 8 bits (mk_kv_append in include/mako_b200.h).
//
// A run is the tokens of a pass that go into one page, rows in order; the CTA that finds a run's first row does all of it for some of
// the heads: the rows' angles once, then for every head the largest key and value, the page's new scales, the codes. A scale is a
// power of two, so that a page whose scale grows (a later token is larger than all before) has its older codes multiplied by a power of
// two, which changes nothing but what becomes subnormal: a token's code does not depend on how often the scale has grown since, and
// dividing by a scale is exact. (A page's scale that somebody else has put there may be another number: quotients are rounded to fp32 then.)
//
// Angles are formed and brought into [-pi, pi] in 64 bits (position x frequency in 32 bits is off by 0.06 rad at a million), their sine and
// cosine in 32, with what an angle loses by its own rounding added.
//
// 64 tokens of a decode step take 6.5 us from a graph, 8 key heads of 128 with 32 query heads; chunks of some 7000 tokens 69, where
// reading and writing once would take 21: instructions bound it, of angles (a third) and of roundings. Two heads a CTA: with one 85 us, whose angles
// are formed eight times, with four 85, too few CTAs.
#include "kv_cache.cuh"
#include "ptx.cuh"
#include "round_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kHeadsEach = 2;    // key heads of a CTA, which share the angles
constexpr uint32_t kTokens = 65536;   // of a run without a rotation at a time, so that its rows' count stays within 31 bits
static_assert((uint64_t)kTokens * kHeadsEach * (2u + kAppendMaxGroup) + kThreads < (1ull << 31), "rows are counted in 31 bits");
constexpr uint32_t kAngles = 4096;    // (cosine, sine) pairs kept for a run's tokens: 32 KB

template <typename T>
__device__ __forceinline__ void load8f(float (&x)[8], const T* p)
{
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 y;
        if constexpr (std::is_same<T, __half>::value)
            y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else
            y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        x[2 * i] = y.x;
        x[2 * i + 1] = y.y;
    }
}

template <typename T>
__device__ __forceinline__ void store8f(T* p, const float (&x)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 y = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&y);
        } else {
            const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&y);
        }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Sixteen columns of a head, the two halves of item j of dim / 16: a pair of the rotation is a[i], b[i] in the half layout, and
// x[2i], x[2i + 1] of the sixteen in the interleaved one; either way frequencies 8j to 8j + 7. Columns behind the rotated ones lie together.
struct Item {
    uint32_t a, b;  // first columns
    uint32_t freq;  // first frequency
    bool turns;
};

__device__ __forceinline__ Item item_of(const KvAppendArgs& a, uint32_t j)
{
    const uint32_t turned = a.rotary / 16u;
    if (j >= turned)
        return Item{16u * j, 16u * j + 8u, 0u, false};
    if (a.interleaved)
        return Item{16u * j, 16u * j + 8u, 8u * j, true};
    return Item{8u * j, a.rotary / 2u + 8u * j, 8u * j, true};
}

__device__ __forceinline__ void turn(float (&x)[8], float (&y)[8], const float2* cs, bool interleaved)
{
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 c = cs[i], d = cs[4 + i];
            const float a0 = x[2 * i], a1 = x[2 * i + 1], b0 = y[2 * i], b1 = y[2 * i + 1];
            x[2 * i] = a0 * c.x - a1 * c.y;
            x[2 * i + 1] = a1 * c.x + a0 * c.y;
            y[2 * i] = b0 * d.x - b1 * d.y;
            y[2 * i + 1] = b1 * d.x + b0 * d.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 c = cs[i];
            const float a = x[i], b = y[i];
            x[i] = a * c.x - b * c.y;
            y[i] = b * c.x + a * c.y;
        }
    }
}

// The largest finite magnitude of eight, as its bits (which are in the order of the numbers).
__device__ __forceinline__ uint32_t largest8(const float (&x)[8], uint32_t m)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
        m = u < 0x7f800000u && u > m ? u : m;
    }
    return m;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const KvAppendArgs a)
{
    __shared__ float2 cs[kAngles];
    __shared__ uint32_t s_most[2 * kHeadsEach];
    __shared__ float s_scale[2 * kHeadsEach], s_old[2 * kHeadsEach];
    __shared__ uint32_t s_len;
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t tid = threadIdx.x, items = a.c.dim / 16u, half = a.rotary / 2u;
    const uint32_t h0 = blockIdx.y * kHeadsEach, heads = min(kHeadsEach, a.c.n_heads - h0);
    const int64_t n_slots = (int64_t)a.c.n_pages * a.c.page_size;
    auto slot_of = [&](uint32_t t) -> int64_t {
        const int64_t x = a.slots[t];
        return x < 0 || x >= n_slots ? -1 : x;
    };
    // A thread has the same columns of all its rows. (Threads that make no whole row of items have none.)
    const uint32_t j = tid % items, step = kThreads / items, row0 = tid / items < step ? tid / items : ~0u >> 1;
    const Item turned = item_of(a, j);
    const uint32_t t_end = min(a.n_tokens, (blockIdx.x + 1u) * a.tokens_each);
    for (uint32_t t0 = blockIdx.x * a.tokens_each; t0 < t_end; ++t0) {
        const int64_t slot = slot_of(t0);
        if (slot < 0)
            continue;
        const uint64_t page = (uint64_t)slot / a.c.page_size;
        const uint32_t place = (uint32_t)((uint64_t)slot - page * a.c.page_size);
        if (place && t0 && slot_of(t0 - 1u) == slot - 1)
            continue; // not a run's first row
        const uint32_t most = min(a.c.page_size - place, a.n_tokens - t0);
        __syncthreads(); // an earlier run is done with what is shared
        if (tid == 0)
            s_len = most;
        if (tid < 2u * kHeadsEach)
            s_most[tid] = 0;
        __syncthreads();
        for (uint32_t i = 1u + tid; i < most; i += kThreads)
            if (a.slots[t0 + i] != slot + i) {
                atomicMin(&s_len, i);
                break;
            }
        __syncthreads();
        const uint32_t len = s_len;
        const uint32_t chunk = min(len, half ? kAngles / half : kTokens); // tokens whose angles are kept at a time
        uint32_t largest[2 * kHeadsEach] = {}; // of keys and values, by head
        for (int pass = 0; pass < 2; ++pass) {
            for (uint32_t i0 = 0; i0 < len; i0 += chunk) {
                const uint32_t n = min(chunk, len - i0);
                if (half && (pass == 0 || chunk < len)) {
                    __syncthreads();
                    for (uint32_t i = tid; i < n * half; i += kThreads) {
                        const uint32_t t = i / half, f = i - t * half;
                        const double x = (double)a.positions[t0 + i0 + t] * (double)__ldg(a.inv_freq + f);
                        const double whole = rint(x * 0.15915494309189533577);
                        const double left = fma(whole, -6.28318530717958647693, x);
                        const float angle = (float)left, rest = (float)(left - angle); // (up to 2^-23 at pi)
                        float sine, cosine;
                        sincosf(angle, &sine, &cosine);
                        cs[i] = make_float2(fmaf(-sine, rest, cosine) * a.rotary_scale, fmaf(cosine, rest, sine) * a.rotary_scale);
                    }
                    __syncthreads();
                }
                // rows of a token: keys and values of these heads and, the first time, the queries that go with them
                const uint32_t rows = 2u * heads + (pass == 0 ? heads * a.group : 0u), all = n * rows;
                uint32_t t = row0 / rows, row = row0 - t * rows;
                for (uint32_t i = row0; i < all; i += step) {
                    const uint64_t token = t0 + i0 + t;
                    const bool query = row >= 2u * heads, value = !query && row >= heads;
                    const uint32_t head = query ? row - 2u * heads : value ? row - heads : row; // among the CTA's
                    const T* p;
                    if (query)
                        p = static_cast<const T*>(a.q) + token * a.q_ld + (uint64_t)(h0 * a.group + head) * a.c.dim;
                    else
                        p = static_cast<const T*>(value ? a.v : a.k) + token * (value ? a.v_ld : a.k_ld) + (uint64_t)(h0 + head) * a.c.dim;
                    const Item at = value ? Item{16u * j, 16u * j + 8u, 0u, false} : turned;
                    float x[8], y[8];
                    load8f(x, p + at.a);
                    load8f(y, p + at.b);
                    if (at.turns)
                        turn(x, y, cs + t * half + at.freq, a.interleaved);
                    const uint32_t which = value ? kHeadsEach + head : head;
                    if (query) {
                        T* to = static_cast<T*>(a.q_out) + token * a.q_out_ld + (uint64_t)(h0 * a.group + head) * a.c.dim;
                        store8f(to + at.a, x);
                        store8f(to + at.b, y);
                    } else if (pass == 0) {
                        const uint32_t m = largest8(y, largest8(x, 0u));
#pragma unroll
                        for (uint32_t k = 0; k < 2u * kHeadsEach; ++k)
                            largest[k] = which == k ? max(largest[k], m) : largest[k];
                    } else {
                        const float scale = s_scale[which];
                        float by = 1.0f / scale;
                        if (__float_as_uint(scale) & 0x7fffffu) { // a page's own, no power of two (the inverse is rounded): quotients
                            by = 1.0f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                x[i] = __fdiv_rn(x[i], scale);
                                y[i] = __fdiv_rn(y[i], scale);
                            }
                        }
                        uint8_t* to = static_cast<uint8_t*>(value ? a.c.v : a.c.k) + page * a.c.page_stride + (uint64_t)(h0 + head) * a.c.head_stride +
                                      (uint64_t)(place + i0 + t) * a.c.token_stride;
                        *reinterpret_cast<uint2*>(to + at.a) = make_uint2(codes4(x, 0, by), codes4(x, 4, by));
                        *reinterpret_cast<uint2*>(to + at.b) = make_uint2(codes4(y, 0, by), codes4(y, 4, by));
                    }
                    row += step;
                    while (row >= rows) {
                        row -= rows;
                        ++t;
                    }
                }
            }
            if (pass)
                break;
            __syncwarp();
#pragma unroll
            for (uint32_t k = 0; k < 2u * kHeadsEach; ++k) {
                const uint32_t m = __reduce_max_sync(~0u, largest[k]);
                if (tid % 32u == 0 && m)
                    atomicMax(&s_most[k], m);
            }
            __syncthreads();
            if (tid < 2u * kHeadsEach && tid % kHeadsEach < heads) {
                const bool value = tid >= kHeadsEach;
                float* at = (value ? a.c.v_scale : a.c.k_scale) + page * a.c.n_heads + h0 + tid % kHeadsEach;
                const float need = scale_of(s_most[tid]), old = place ? *at : 0.0f;
                const float now = old > need ? old : need;
                s_old[tid] = old;
                s_scale[tid] = now;
                *at = now;
            }
            __syncthreads();
            // codes of the tokens that were there before, where their scale has grown
            for (uint32_t which = 0; place && which < 2u * kHeadsEach; ++which) {
                if (which % kHeadsEach >= heads || s_old[which] == s_scale[which])
                    continue;
                const float by = s_old[which] / s_scale[which];
                uint8_t* p = static_cast<uint8_t*>(which >= kHeadsEach ? a.c.v : a.c.k) + page * a.c.page_stride +
                             (uint64_t)(h0 + which % kHeadsEach) * a.c.head_stride;
                for (uint32_t i = tid; i < place * items; i += kThreads) {
                    uint4* q = reinterpret_cast<uint4*>(p + (uint64_t)(i / items) * a.c.token_stride + i % items * 16u);
                    const uint4 x = *q;
                    *q = make_uint4(rescale4(x.x, by), rescale4(x.y, by), rescale4(x.z, by), rescale4(x.w, by));
                }
            }
        }
    }
}

} // namespace

cudaError_t launch_kv_append(const KvAppendArgs& args, int type, cudaStream_t stream)
{
    KvAppendArgs a = args;
    a.tokens_each = a.n_tokens <= 1024u ? 1u : 16u;
    const dim3 grid((a.n_tokens + a.tokens_each - 1) / a.tokens_each, (a.c.n_heads + kHeadsEach - 1) / kHeadsEach);
    if (type == MK_BF16)
        kv_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(a);
    else
        kv_append_kernel<__half><<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

} // namespace mk
