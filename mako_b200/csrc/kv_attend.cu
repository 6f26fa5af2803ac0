// Attention of few rows over a paged 8-bit cache (mk_kv_attention in include/mako_b200.h): a decode step, a speculative round. Every
// key and value is read once for 16 rows, tokens of the pass times query heads that share the key head, and from L2 for 16 more. HBM bounds
// it where contexts are long (64 sequences of up to 16384 keys, 8 key heads of 128, 4 query heads each: 183 us for 987 MB, 5.4 TB/s or 0.82 of the
// rate of a copy; two of 131072 with groups of 8: 107 us, 0.77), latency where they are short (one sequence of 2048: 14.5 us from a graph, of which the
// search for a CTA's share is 1.6, the chain from page to product 2, the join 5).
//
// A unit has 16 rows: the MMA's M. A warp takes every fourth block of its CTA's keys, 32 keys and values (8 KB at 128 columns), which it
// copies into a ring of its own in shared memory, so that warps wait for nobody until their segment ends; three CTAs of four warps an SM,
// two blocks each, have 98 KB under way. (When it took 195 us: with blocks of 16 keys, four deep, 214, 1.3 times the instructions; with two CTAs
// and three blocks 218, too few warps for the chain of product, exponential, product. Two tiles of rows that share what is read had 32 rows take 113 us
// where two units take 129, but 24 rows 194 against 163.)
// mma.sync, not tcgen05: 16 rows are an eighth of that one's M, and a product's operands would have to go through shared memory as fp16, which
// is four times the bytes that the cache's codes are there. The tensor pipe is busy for 0.35 of the time.
//
// Codes become fp16 (exactly) on the way from shared memory into registers, in the order in which the tensor core wants them: of a block's
// keys a lane reads 16 of a token's columns, four steps of the contraction; of its values the four tokens whose weights it holds, which
// byte permutations put side by side. Queries are fp16 too, each row times the power of two that brings its largest to about 2^12: bf16 loses
// nothing by it down to 2^-29 of that one. Scales of keys go into the scores, scales of values into the weights, which fp16 holds in a unit of the row's own (kv_unit in
// kv_work.cuh); sums are in fp32.
#include "kv_cache.cuh"
#include "kv_work.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

namespace mk {
namespace {

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kStages = 2;
constexpr uint32_t kTile = 16, kBlockTokens = 32; // rows of a unit, keys of a block

template <uint32_t D>
constexpr uint32_t kStageBytes = 2 * kBlockTokens * (D + 4); // keys and values, two scales a token
template <uint32_t D>
constexpr uint32_t kRingBytes = kStages * kStageBytes<D>;

__device__ __forceinline__ void copy16(void* to, const void* from, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from, bool there)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <uint32_t N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pair_of(float x, float y)
{
    const __half2 r = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Where the 16 bytes `chunk` of a token's keys, and of its values, lie in a block: such that the lanes that read at the same time
// (keys: two tokens' four chunks; values: every second token's same chunk) are in different banks.
template <uint32_t D>
__device__ __forceinline__ uint32_t key_at(uint32_t token, uint32_t chunk)
{
    return D == 128 ? token * 128u + ((chunk ^ ((token & 1u) << 2)) << 4) : token * 64u + (chunk << 4);
}
template <uint32_t D>
__device__ __forceinline__ uint32_t value_at(uint32_t token, uint32_t chunk)
{
    return D == 128 ? token * 128u + ((chunk ^ (token & 7u)) << 4)
                    : (token >> 1) * 128u + (((((token & 1u) << 2) + chunk) ^ ((token & 6u))) << 4);
}

template <uint32_t D>
struct Shared {
    uint64_t find[40];
    float factor[kTile];               // of a row's scores
    int32_t lo[kTile], hi[kTile];    // the keys that a row sees: [lo, hi)
    float m[kWarps][kTile], l[kWarps][kTile];
    uint32_t valid[kWarps][kStages];
    uint4 q[D / 16 * 32];         // queries in the order of the MMA's registers
};

template <typename T>
__device__ __forceinline__ float2 two(uint32_t w)
{
    if constexpr (std::is_same<T, __half>::value)
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The unit's queries: a thread has 16 columns of a row.
template <typename T, uint32_t D>
__device__ void load_queries(const KvAttendArgs& a, Shared<D>& s, const KvSegment& u)
{
    constexpr uint32_t chunks = D / 16;
    for (uint32_t i = threadIdx.x; i < kTile * chunks; i += kThreads) { // (whole warps: chunks divides 32)
        const uint32_t r = i / chunks, chunk = i % chunks, row = u.row0 + r;
        const bool real = r < u.rows;
        const uint32_t token = kv_token_of(a, row);
        uint32_t w[8] = {};
        if (real) {
            const T* p = static_cast<const T*>(a.q) + (u.seq.first + token) * a.q_ld + (uint64_t)(u.head * a.group + row - token * a.group) * D + chunk * 16u;
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p)), y = __ldg(reinterpret_cast<const uint4*>(p) + 1);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
        }
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 x = two<T>(w[k]);
            most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
#pragma unroll
        for (uint32_t d = 1; d < chunks; d <<= 1)
            most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
        // a power of two, from 2^-115; 1 where a row is nothing or infinite
        const int e = (int)(__float_as_uint(most) >> 23) - 127;
        const int up = most > 0.0f && e < 128 ? min(100, 12 - e) : 0;
        const float by = __uint_as_float((uint32_t)(up + 127) << 23);
        uint32_t* to = reinterpret_cast<uint32_t*>(s.q) + (chunk / 4u * 128u + (r & 7u) * 4u + (chunk & 3u)) * 4u + (r >> 3);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) { // a step of the contraction each
            const float2 x = two<T>(w[2 * k]), y = two<T>(w[2 * k + 1]);
            to[k * 128u] = pair_of(x.x * by, x.y * by);
            to[k * 128u + 2u] = pair_of(y.x * by, y.y * by);
        }
        if (chunk == 0) {
            const int64_t at = (int64_t)u.seq.len - u.seq.n + token; // its position
            s.factor[r] = a.scale_log2 / by;
            s.hi[r] = real && at >= 0 ? (int32_t)(at + 1 < u.seq.keys ? at + 1 : u.seq.keys) : 0;
            s.lo[r] = a.window && at + 1 > (int64_t)a.window ? (int32_t)(at + 1 - a.window) : 0;
        }
    }
}

// A warp's copies of blocks of keys and values. 16 tokens are looked up at a time where pages are a multiple of that, else each by itself.
template <uint32_t D>
struct Copier {
    static constexpr uint32_t tokens = kBlockTokens, row_chunks = D / 16, rows_each = 32 / row_chunks;
    const KvAttendArgs* a;
    unsigned char* ring;
    uint32_t* valid;              // a bit for each token of a stage's block: it is there
    const int32_t* table;
    uint32_t keys, head;
    bool wide;                    // is a page a multiple of 16 tokens?

    // The page of this lane's token of a block, early: what it is good for is issued when it is there.
    __device__ __forceinline__ int32_t look_up(uint32_t block) const
    {
        const uint32_t t = block * tokens + (threadIdx.x & 31u);
        return t < keys ? __ldg(table + kv_page_of(*a, t)) : -1;
    }
    __device__ __forceinline__ void issue(uint32_t block, uint32_t stage, int32_t page) const
    {
        const uint32_t lane = threadIdx.x & 31u, t = block * tokens + lane;
        unsigned char* to = ring + stage * kStageBytes<D>;
        const bool there = (uint32_t)page < a->c.n_pages;
        const uint32_t p = there ? (uint32_t)page : 0u;
        const uint32_t mask = __ballot_sync(~0u, there);
        float* scales = reinterpret_cast<float*>(to + 2 * tokens * D);
        const uint64_t at = (uint64_t)p * a->c.n_heads + head;
        copy4(scales + lane, a->c.k_scale + at, there);
        copy4(scales + tokens + lane, a->c.v_scale + at, there);
        if (lane == 0)
            valid[stage] = mask;
        const uint32_t chunk = lane % row_chunks, row = lane / row_chunks;
        const uint64_t stride = a->c.token_stride;
        if (wide) {
#pragma unroll
            for (uint32_t h = 0; h < tokens / 16u; ++h) { // a page's part
                const uint32_t first = block * tokens + 16u * h, its = __shfl_sync(~0u, p, 16u * h);
                const uint64_t base = (uint64_t)its * a->c.page_stride + (uint64_t)head * a->c.head_stride + chunk * 16u +
                                      (uint64_t)(first - kv_page_of(*a, first) * a->c.page_size + row) * stride;
                const unsigned char *k = static_cast<const unsigned char*>(a->c.k) + base, *v = static_cast<const unsigned char*>(a->c.v) + base;
#pragma unroll
                for (uint32_t i = 0; i < 16u / rows_each; ++i) {
                    const uint32_t r = 16u * h + i * rows_each + row;
                    const bool ok = (mask >> r) & 1u;
                    copy16(to + key_at<D>(r, chunk), k, ok);
                    copy16(to + tokens * D + value_at<D>(r, chunk), v, ok);
                    k += rows_each * stride;
                    v += rows_each * stride;
                }
            }
        } else {
            const uint32_t place = there ? t - kv_page_of(*a, t) * a->c.page_size : 0u;
            const uint64_t off = (uint64_t)p * a->c.page_stride + (uint64_t)head * a->c.head_stride + (uint64_t)place * stride;
#pragma unroll
            for (uint32_t i = 0; i < tokens / rows_each; ++i) {
                const uint32_t r = i * rows_each + row;
                const uint64_t from = __shfl_sync(~0u, off, r) + chunk * 16u;
                const bool ok = (mask >> r) & 1u;
                copy16(to + key_at<D>(r, chunk), static_cast<const unsigned char*>(a->c.k) + from, ok);
                copy16(to + tokens * D + value_at<D>(r, chunk), static_cast<const unsigned char*>(a->c.v) + from, ok);
            }
        }
    }
};

// What a warp has of a unit: rows g and g + 8 of each tile (g: its lane / 4) and, of them, 2 * D / 8 columns.
template <uint32_t D>
struct Running {
    float m[2], l[2], o[D / 8][4];
    float factor[2];
    float unit[2]; // see kv_unit
};

// Is one of four codes NaN? And the codes without those.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

template <uint32_t D>
__device__ __forceinline__ void add_block(Running<D>& x, const Shared<D>& s, const unsigned char* stage, uint32_t valid, uint32_t block, bool all_see)
{
    constexpr uint32_t tokens = kBlockTokens, NT = tokens / 8, words = D / 32;
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, c = lane & 3u;
    const float* scales = reinterpret_cast<const float*>(stage + 2 * tokens * D);
    float t[NT][4] = {};
#pragma unroll
    for (uint32_t h = 0; h < D / 64; ++h) {
        uint4 w[NT];
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
            w[n] = *reinterpret_cast<const uint4*>(stage + key_at<D>(n * 8u + g, c + 4u * h));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint4 q = s.q[(h * 4u + i) * 32u + lane];
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                const uint2 b = halves_of4(i == 0 ? w[n].x : i == 1 ? w[n].y : i == 2 ? w[n].z : w[n].w);
                mma16(t[n], q, b.x, b.y);
            }
        }
    }
    float2 vs[NT];
    float v_most = 0.0f;
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        const float2 ks = *reinterpret_cast<const float2*>(scales + n * 8u + 2u * c);
        vs[n] = *reinterpret_cast<const float2*>(scales + tokens + n * 8u + 2u * c);
        v_most = fmaxf(v_most, fmaxf(vs[n].x, vs[n].y));
        t[n][0] *= ks.x * x.factor[0];
        t[n][1] *= ks.y * x.factor[0];
        t[n][2] *= ks.x * x.factor[1];
        t[n][3] *= ks.y * x.factor[1];
    }
    v_most = fmaxf(v_most, __shfl_xor_sync(~0u, v_most, 1));
    v_most = fmaxf(v_most, __shfl_xor_sync(~0u, v_most, 2));
    auto sees = [&](uint32_t n, uint32_t e) {
        const uint32_t j = n * 8u + 2u * c + (e & 1u), r = g + (e >> 1) * 8u;
        const int32_t key = (int32_t)(block * tokens + j);
        return ((valid >> j) & 1u) && key >= s.lo[r] && key < s.hi[r];
    };
    if (!all_see) {
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (!sees(n, e))
                    t[n][e] = -INFINITY;
    }
    float from[2];
    bool grows = false; // may a row's unit have to grow? By the largest scale of all these keys, seen or not: whether it does is looked up below
    const float v_log = __log2f(v_most);
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
        float most = -INFINITY;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
            most = fmaxf(most, fmaxf(t[n][2 * r], t[n][2 * r + 1]));
        most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
        most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
        const float m = fmaxf(x.m[r], most);
        from[r] = m == -INFINITY ? 0.0f : m;
        const float by = ex2_approx(x.m[r] - from[r]);
        x.m[r] = m;
        float l = 0.0f;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) {
            const float a = ex2_approx(t[n][2 * r] - from[r]), b = ex2_approx(t[n][2 * r + 1] - from[r]);
            l += a + b;
            const float2 w = mul2(make_float2(a, b), vs[n]);
            t[n][2 * r] = w.x;
            t[n][2 * r + 1] = w.y;
        }
        x.l[r] = x.l[r] * by + l;
        grows = grows || kv_unit(x.unit[r], most + v_log, from[r]) != x.unit[r];
    }
    if (__any_sync(~0u, grows)) {
        float older[2]; // what outputs so far are worth
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r) {
            float top = 0.0f;
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
                top = fmaxf(top, fmaxf(t[n][2 * r], t[n][2 * r + 1]));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            const float unit = kv_unit(x.unit[r], from[r] + __log2f(top), from[r]);
            older[r] = unit == x.unit[r] ? 1.0f : kv_worth(x.unit[r], unit);
            x.unit[r] = unit;
        }
#pragma unroll
        for (uint32_t j = 0; j < D / 8; ++j) {
            x.o[j][0] *= older[0];
            x.o[j][1] *= older[0];
            x.o[j][2] *= older[1];
            x.o[j][3] *= older[1];
        }
    }
    uint4 p[NT / 2];
    const float e0 = ex2_approx(from[0] - x.unit[0]), e1 = ex2_approx(from[1] - x.unit[1]);
    const float2 by0 = make_float2(e0, e0), by1 = make_float2(e1, e1);
#pragma unroll
    for (uint32_t n = 0; n < NT; n += 2) {
        const float2 w0 = mul2(make_float2(t[n][0], t[n][1]), by0), w1 = mul2(make_float2(t[n][2], t[n][3]), by1);
        const float2 w2 = mul2(make_float2(t[n + 1][0], t[n + 1][1]), by0), w3 = mul2(make_float2(t[n + 1][2], t[n + 1][3]), by1);
        p[n / 2] = make_uint4(pair_of(w0.x, w0.y), pair_of(w1.x, w1.y), pair_of(w2.x, w2.y), pair_of(w3.x, w3.y));
    }
    const unsigned char* values = stage + tokens * D;
#pragma unroll
    for (uint32_t k = 0; k < NT / 2; ++k) {
        uint32_t w[4][words];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t token = k * 16u + 2u * c + (i & 1u) + (i >> 1) * 8u;
            if constexpr (D == 128) {
                const uint4 y = *reinterpret_cast<const uint4*>(values + value_at<D>(token, g));
                w[i][0] = y.x, w[i][1] = y.y, w[i][2] = y.z, w[i][3] = y.w;
            } else {
                const uint2 y = *reinterpret_cast<const uint2*>(values + value_at<D>(token, g >> 1) + (g & 1u) * 8u);
                w[i][0] = y.x, w[i][1] = y.y;
            }
        }
        if (!all_see) { // a weight of nothing times NaN would be NaN: rows that see such a value are, the others are not to be
            uint32_t bad = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t j = 0; j < words; ++j)
                    bad |= nan_bytes(w[i][j]) ? 1u << i : 0u;
            if (__any_sync(~0u, bad)) {
                bad |= __shfl_xor_sync(~0u, bad, 4);
                bad |= __shfl_xor_sync(~0u, bad, 8);
                bad |= __shfl_xor_sync(~0u, bad, 16);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
#pragma unroll
                    for (uint32_t j = 0; j < words; ++j)
                        w[i][j] &= ~nan_bytes(w[i][j]);
#pragma unroll
                    for (uint32_t r = 0; r < 2; ++r)
                        if ((bad >> i & 1u) && sees(2u * k + (i >> 1), 2u * r + (i & 1u)))
                            x.l[r] = __int_as_float(0x7fc00000);
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < words; ++j) {
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                const uint32_t order = half ? 0x7362u : 0x5140u; // two tokens' codes of a column side by side
                const uint2 b0 = halves_of4(__byte_perm(w[0][j], w[1][j], order)), b1 = halves_of4(__byte_perm(w[2][j], w[3][j], order));
                mma16(x.o[4u * j + 2u * half], p[k], b0.x, b1.x);
                mma16(x.o[4u * j + 2u * half + 1u], p[k], b0.y, b1.y);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float4& x)
{
    uint2 r;
    if constexpr (std::is_same<T, __half>::value) {
        r = make_uint2(pair_of(x.x, x.y), pair_of(x.z, x.w));
    } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y), z = __floats2bfloat162_rn(x.z, x.w);
        r = make_uint2(*reinterpret_cast<const uint32_t*>(&y), *reinterpret_cast<const uint32_t*>(&z));
    }
    *reinterpret_cast<uint2*>(p) = r;
}

// A row's place in the output.
template <typename T, uint32_t D>
__device__ __forceinline__ T* out_row(const KvAttendArgs& a, const KvSegment& u, uint32_t r)
{
    const uint32_t row = u.row0 + r;
    const uint32_t token = kv_token_of(a, row);
    return static_cast<T*>(a.out) + (u.seq.first + token) * a.out_ld + (uint64_t)(u.head * a.group + row - token * a.group) * D;
}

__device__ __forceinline__ float part_factor(float m, float most) { return m == -INFINITY ? 0.0f : ex2_approx(m - most); }
__device__ __forceinline__ void add4(float4& x, const float4& y, float by)
{
    x.x += y.x * by;
    x.y += y.y * by;
    x.z += y.z * by;
    x.w += y.w * by;
}
__device__ __forceinline__ float4 over(const float4& x, float l) // a row that saw nothing is zeros
{
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    return make_float4(x.x * by, x.y * by, x.z * by, x.w * by);
}

template <uint32_t D>
constexpr uint32_t kPartFloats = kTile * (D + 2u); // outputs, maxima, sums

template <typename T, uint32_t D>
__global__ void __launch_bounds__(kThreads, 3) kv_rows_kernel(const KvAttendArgs a)
{
    extern __shared__ __align__(128) unsigned char raw[]; // the warps' rings; behind a segment, what they have of it
    __shared__ Shared<D> s;
    constexpr uint32_t tile = kTile, each = kBlockTokens, row_floats = D + 4;
    const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid & 31u, g = lane >> 2, c = lane & 3u;
    griddep_launch_dependents();
    griddep_wait();
    KvWalk walk = kv_find<kThreads>(a, tile, each, gridDim.x, s.find, blockIdx.x);
    Copier<D> copier;
    copier.a = &a;
    copier.ring = raw + warp * kRingBytes<D>;
    copier.valid = s.valid[warp];
    copier.wide = a.c.page_size % 16u == 0;
    KvSegment u;
    for (bool first = true; kv_take(a, walk, u, first, tile, each); first = false) {
        const uint32_t from = u.from, to = u.to;
        copier.table = a.block_table + (uint64_t)u.sq * a.table_ld;
        copier.keys = u.seq.keys;
        copier.head = u.head;
        uint32_t next = from + warp;
        int32_t pages[kStages];
#pragma unroll
        for (uint32_t i = 0; i < kStages; ++i)
            pages[i] = next + i * kWarps < to ? copier.look_up(next + i * kWarps) : -1;
#pragma unroll
        for (uint32_t i = 0; i + 1 < kStages; ++i, next += kWarps) {
            if (next < to)
                copier.issue(next, i, pages[i]);
            copies_close();
        }
        int32_t page = pages[kStages - 1];
        load_queries<T, D>(a, s, u);
        __syncthreads();
        const uint32_t see_from = (uint32_t)s.lo[u.rows - 1u], see_to = (uint32_t)s.hi[0];
        Running<D> x;
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r) {
            x.factor[r] = s.factor[g + 8u * r];
            x.unit[r] = INFINITY;
            x.m[r] = -INFINITY;
            x.l[r] = 0.0f;
        }
#pragma unroll
        for (uint32_t j = 0; j < D / 8; ++j)
            x.o[j][0] = x.o[j][1] = x.o[j][2] = x.o[j][3] = 0.0f;
        uint32_t stage = 0;
        for (uint32_t block = from + warp; block < to; block += kWarps, next += kWarps) {
            if (next < to) {
                copier.issue(next, stage == 0 ? kStages - 1u : stage - 1u, page);
                page = copier.look_up(next + kWarps);
            }
            copies_close();
            copies_wait<kStages - 1>();
            __syncwarp();
            const uint32_t valid = s.valid[warp][stage];
            const bool all_see = valid == ~0u && block * each >= see_from && (block + 1u) * each <= see_to;
            add_block<D>(x, s, copier.ring + stage * kStageBytes<D>, valid, block, all_see);
            __syncwarp();
            stage = stage + 1u == kStages ? 0u : stage + 1u;
        }
        copies_wait<0>();
        __syncthreads();
        float* mine = reinterpret_cast<float*>(raw + warp * kRingBytes<D>);
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r) {
            const float worth = kv_worth(x.unit[r], x.m[r]);
            float l = x.l[r];
            l += __shfl_xor_sync(~0u, l, 1);
            l += __shfl_xor_sync(~0u, l, 2);
            const uint32_t row = r * 8u + g;
            if (c == 0) {
                s.m[warp][row] = x.m[r];
                s.l[warp][row] = l;
            }
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e)
#pragma unroll
                for (uint32_t j = 0; j < D / 8; j += 4)
                    *reinterpret_cast<float4*>(mine + row * row_floats + (2u * c + e) * (D / 8) + j) =
                        make_float4(x.o[j][2 * r + e] * worth, x.o[j + 1][2 * r + e] * worth, x.o[j + 2][2 * r + e] * worth, x.o[j + 3][2 * r + e] * worth);
        }
        __syncthreads();
        const bool whole = u.whole();
        float* part = a.parts + (uint64_t)u.place(blockIdx.x) * kPartFloats<D>;
        for (uint32_t i = tid; i < u.rows * (D / 4); i += kThreads) {
            const uint32_t r = i / (D / 4), d = i % (D / 4) * 4u;
            float most = s.m[0][r];
#pragma unroll
            for (uint32_t w = 1; w < kWarps; ++w)
                most = fmaxf(most, s.m[w][r]);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float l = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float f = part_factor(s.m[w][r], most);
                l += s.l[w][r] * f;
                add4(o, *reinterpret_cast<const float4*>(raw + w * kRingBytes<D> + (r * row_floats + d) * 4u), f);
            }
            if (whole) {
                store4(out_row<T, D>(a, u, r) + d, over(o, l));
            } else {
                *reinterpret_cast<float4*>(part + r * D + d) = o;
                if (d == 0) {
                    part[tile * D + r] = most;
                    part[tile * (D + 1u) + r] = l;
                }
            }
        }
        __syncthreads(); // before the next segment's copies, queries and limits
    }
}

// Puts the units together that a cut goes through, a CTA for each cut: the first one inside a unit does it.
constexpr uint32_t kJoinThreads = 256, kJoinParts = 32;

template <typename T, uint32_t D, uint32_t Tile, uint32_t Each>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttendArgs a, const uint32_t ctas_most)
{
    __shared__ uint64_t scratch[40];
    __shared__ float s_factor[kJoinParts][16], s_by[16];
    const uint32_t cta = blockIdx.x + 1u, tid = threadIdx.x;
    KvWalk walk = kv_find<kJoinThreads>(a, Tile, Each, ctas_most, scratch, cta); // (from what was there before the units were begun)
    griddep_wait(); // (by those that have nothing to do too: what follows waits for this launch)
    if (cta >= walk.ctas)
        return;
    const uint32_t skip = walk.skip, ctas = walk.ctas;
    const uint64_t start = walk.at - skip;
    if (skip == 0 || kv_cut(walk.total, ctas, cta - 1u) > start)
        return;
    KvSegment u;
    u.from = u.to = 0;
    u.blocks = KvBlocks{0, 0};
    kv_take(a, walk, u, true, Tile, Each);
    const uint32_t blocks = u.blocks.to - u.blocks.from;
    if (skip >= blocks || u.from != u.blocks.from + skip) // the cut is behind the unit's blocks (and what was taken is another one's)
        return;
    const uint64_t stop = start + blocks;
    constexpr uint32_t floats = Tile * (D + 2u);
    uint32_t parts = 1; // of the CTA that began the unit, and of those whose shares begin inside
    while (cta + parts - 1u < ctas && kv_cut(walk.total, ctas, cta + parts - 1u) < stop)
        ++parts;
    auto join_row = [](uint32_t i) { return Tile > 32 ? i % 16u : i / (D / 4); };
    auto join_column = [](uint32_t i) { return (Tile > 32 ? i / 16u : i % (D / 4)) * 4u; };
    auto part = [&](uint32_t p) { return a.parts + (uint64_t)(2u * (cta - 1u + p) + (p == 0)) * floats; };
    for (uint32_t r0 = 16u * blockIdx.y; r0 < u.rows; r0 += 16u * gridDim.y) { // 16 rows at a time: their maxima, then what each part is worth, then the sums
        const uint32_t rows = min(16u, u.rows - r0);
        float4 o[16 * (D / 4) / kJoinThreads];
#pragma unroll
        for (uint32_t k = 0; k < 16 * (D / 4) / kJoinThreads; ++k)
            o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f, most = -INFINITY;
        // (a row's maximum over all parts first: by the 16 threads that share its row, through shuffles)
        const uint32_t row = tid / 16u, lane = tid % 16u;
        if (row < rows)
            for (uint32_t p = lane; p < parts; p += 16u)
                most = fmaxf(most, part(p)[Tile * D + r0 + row]);
        __syncwarp();
#pragma unroll
        for (uint32_t d = 8; d; d >>= 1)
            most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
        for (uint32_t p0 = 0; p0 < parts; p0 += kJoinParts) {
            const uint32_t some = min(kJoinParts, parts - p0);
            __syncthreads();
            if (row < rows)
                for (uint32_t p = lane; p < some; p += 16u) {
                    const float* x = part(p0 + p) + r0 + row;
                    const float f = part_factor(x[Tile * D], most);
                    s_factor[p][row] = f;
                    l += x[Tile * (D + 1u)] * f;
                }
            __syncthreads();
#pragma unroll
            for (uint32_t k = 0; k < 16 * (D / 4) / kJoinThreads; ++k) {
                const uint32_t i = tid + k * kJoinThreads, r = join_row(i), d = join_column(i);
                if (r < rows) {
#pragma unroll 4
                    for (uint32_t p = 0; p < some; ++p) {
                        const float* x = part(p0 + p);
                        float4 y;
                        if constexpr (Tile > 32) { // by column, as kv_prompt_kernel writes them
                            x += d * Tile + r0 + r;
                            y = make_float4(x[0], x[Tile], x[2 * Tile], x[3 * Tile]);
                        } else {
                            y = *reinterpret_cast<const float4*>(x + (r0 + r) * D + d);
                        }
                        add4(o[k], y, s_factor[p][r]);
                    }
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (uint32_t d = 8; d; d >>= 1)
            l += __shfl_xor_sync(~0u, l, d);
        if (lane == 0 && row < rows)
            s_by[row] = l;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < 16 * (D / 4) / kJoinThreads; ++k) {
            const uint32_t i = tid + k * kJoinThreads, r = join_row(i), d = join_column(i);
            if (r < rows)
                store4(out_row<T, D>(a, u, r0 + r) + d, over(o[k], s_by[r]));
        }
        __syncthreads();
    }
}

constexpr uint32_t kRowsCtas = 148u * 3u; // all of which run at the same time
constexpr uint64_t kv_rows_parts(uint32_t dim) { return (uint64_t)kRowsCtas * 2u * kTile * (dim + 2u) * 4u; } // bytes

template <typename T, uint32_t D, uint32_t Tile, uint32_t Each>
cudaError_t launch_join(const KvAttendArgs& a, uint32_t ctas, cudaStream_t stream)
{
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(ctas - 1u, Tile > 64u ? Tile / 64u : 1u); // (all of which run at the same time)
    c.blockDim = dim3(kJoinThreads);
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kv_join_kernel<T, D, Tile, Each>, a, ctas);
}

template <typename T, uint32_t D>
cudaError_t launch_rows(const KvAttendArgs& a, cudaStream_t stream)
{
    constexpr uint32_t smem = kWarps * kRingBytes<D>, grid = kRowsCtas;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = set_once(done, kv_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess)
        return e;
    kv_rows_kernel<T, D><<<grid, kThreads, smem, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess)
        return e;
    return launch_join<T, D, kTile, kBlockTokens>(a, grid, stream);
}

// Sequences of up to so many rows go through kv_rows_kernel, in a pass with longer ones too: it takes the time of as many tiles of 16, a unit of
// kv_prompt_kernel that of 256 rows. 64 sequences of 8192 keys, 8 key heads of 128, by the one and by the other: 48 rows 551 and 730 us, 64 rows
// 762 and 726; 96 rows 1134 and 731.
constexpr uint32_t kFewRows = 64;

template <typename T, uint32_t D>
cudaError_t launch(const KvAttendArgs& args, int type, cudaStream_t stream)
{
    KvAttendArgs a = args;
    const bool few = (uint64_t)a.max_new * a.group <= kFewRows;
    a.rows_from = 1;
    a.rows_to = few ? 0xffffffffu : kFewRows; // (max_new is what the caller says: where it is too small all the same rows are done)
    a.unit_cost = 8; // (4: 187 us where 8 takes 183 and 12 184; 37 sequences of up to 6000, 27, 25, 25)
    a.blocks_least = 8;
    cudaError_t e = launch_rows<T, D>(a, stream);
    if (e != cudaSuccess || few)
        return e;
    a.parts = args.parts + kv_rows_parts(D) / 4u;
    a.rows_from = kFewRows + 1u;
    a.rows_to = 0xffffffffu;
    a.unit_cost = 4; // (0: 1303 us where 4 takes 1295 and 8 1297; chunks of 400 beside 21 single tokens, 121, 95, 97)
    a.blocks_least = 1;
    e = launch_kv_prompt(a, type, stream);
    return e != cudaSuccess ? e : launch_join<T, D, kPromptRows, kPromptBlock>(a, kPromptCtas, stream);
}

} // namespace

uint64_t kv_attend_bytes(uint32_t dim, uint64_t most_rows)
{
    return kv_rows_parts(dim) + (most_rows > kFewRows ? (uint64_t)kPromptCtas * 2u * kPromptRows * (dim + 2u) * 4u : 0u);
}

cudaError_t launch_kv_attend(const KvAttendArgs& a, int type, cudaStream_t stream)
{
    if (type == MK_BF16)
        return a.c.dim == 128u ? launch<__nv_bfloat16, 128>(a, type, stream) : launch<__nv_bfloat16, 64>(a, type, stream);
    return a.c.dim == 128u ? launch<__half, 128>(a, type, stream) : launch<__half, 64>(a, type, stream);
}

} // namespace mk
