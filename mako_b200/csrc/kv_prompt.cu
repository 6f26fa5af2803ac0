// Attention of many rows over a paged 8-bit cache (mk_kv_attention in include/mako_b200.h): prompts' chunks. Here the tensor core bounds, with
// the exponentials beside it: a block of 128 keys past 256 rows of 128 columns is 2048 cycles of either.
//
// A unit has 256 rows, two tiles of the MMA's M, that take turns: while one tile's scores become weights, the tensor core works for the
// other. One warp issues; four (a row of a tile a thread) turn scores into weights, four more for the other tile; four turn the cache's codes
// into fp16, K-major for the keys, the same bytes read as MN-major for the values. Scores and outputs are in tensor memory; weights take
// the scores' place, as the A operand of the second product. An output is multiplied only where a row's maximum has grown by more than
// 2^8, or the largest scale of values.
#include "kv_cache.cuh"
#include "kv_work.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>

namespace mk {
namespace {

constexpr uint32_t kTileRows = 128, kUnitRows = 256, kBlock = 128; // rows of a tile, of a unit; keys of a block
constexpr uint32_t kThreads = 512;
constexpr uint32_t kConvert = 256, kIssue = 384; // first thread of those that convert, and of the warp that issues
constexpr uint32_t kSlots = 4;                   // of what softmax reads beside the scores
constexpr float kWeightUnit = 128.0f;
constexpr uint32_t kMixed = 8; // blocks of a segment that some rows see and others do not: at most 3 at either end

struct Scale {
    float key, value; // the value's: over the largest so far, times kWeightUnit
};

struct Shared {
    uint64_t find[40];
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int failed;
    float factor[kUnitRows];
    int32_t lo[kUnitRows], hi[kUnitRows];
    alignas(16) Scale scale[kSlots][kBlock];
    uint32_t missing[kSlots][4];       // tokens whose page is not there
    float older[kSlots];               // what outputs so far are worth in the block's unit
    float unit[2];                     // the largest scale of a segment's values, by its parity
    uint32_t n_mixed[2];
    uint32_t mixed[2][kMixed][5];      // a block and which of its values are NaN
    uint64_t off[2][kBlock];
    float warp_most[4];
};

__device__ __forceinline__ bool await(Shared& s, uint64_t* bar, uint32_t parity)
{
    if (mbar_try(bar, parity))
        return true;
    const long long from = clock64();
    do {
        if (mbar_try(bar, parity))
            return true;
    } while (clock64() - from < (1ll << 32) && !*reinterpret_cast<volatile int*>(&s.failed));
    *reinterpret_cast<volatile int*>(&s.failed) = 1;
    return false;
}

// D [128 x n] (+)= A [128 x 16] (fp16, in tensor memory) B [16 x n] (fp16, MN-major).
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}

// The same bytes that smem_tile_desc describes, read with the contracted dimension going from row to row: 64 columns side by side, `next`
// bytes to the next 64, 1024 bytes from eight rows to the next.
__device__ __forceinline__ uint64_t smem_rows_desc(const void* tile, uint32_t next)
{
    return (uint64_t)((smem_u32(tile) & 0x3ffffu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

#define MK_R8(x, i) "=f"(x[i]), "=f"(x[i + 1]), "=f"(x[i + 2]), "=f"(x[i + 3]), "=f"(x[i + 4]), "=f"(x[i + 5]), "=f"(x[i + 6]), "=f"(x[i + 7])
#define MK_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])

// 32 columns of this warp's lanes, there when it returns.
__device__ __forceinline__ void tmem_read32(float* x, uint32_t at)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : MK_R8(x, 0), MK_R8(x, 8), MK_R8(x, 16), MK_R8(x, 24)
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_write32(uint32_t at, const uint32_t* x)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31};" ::MK_W8(x, 0),
        MK_W8(x, 8), MK_W8(x, 16), MK_W8(x, 24), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_written() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pair_of(float x, float y)
{
    const __half2 r = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__device__ __forceinline__ float2 two(uint32_t w)
{
    if constexpr (std::is_same<T, __half>::value)
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Where the 16 bytes `chunk` (8 fp16 columns) of a row lie in a tile of 128 rows: 64 columns side by side, 16 KB to the next 64.
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t chunk) { return (chunk >> 3) * 16384u + row * 128u + (((chunk ^ row) & 7u) << 4); }

// A segment: blocks [from, to) of a unit.
struct Segment {
    KvSeq seq;
    KvUnit u;
    uint32_t sq, from, to;
    uint32_t see_from, see_to; // what all rows see
};

template <uint32_t D>
struct Ring { // shared memory
    static constexpr uint32_t tile_bytes = kTileRows * D * 2;
    unsigned char* base;
    __device__ __forceinline__ unsigned char* q(uint32_t t) const { return base + t * tile_bytes; }
    __device__ __forceinline__ unsigned char* k(uint32_t i) const { return base + (2u + i) * tile_bytes; }
    __device__ __forceinline__ unsigned char* v(uint32_t i) const { return base + (4u + i) * tile_bytes; }
};

// Those that convert. What they count goes on from segment to segment.
template <typename T, uint32_t D>
struct Converter {
    static constexpr uint32_t chunks = D / 16, rows_each = 128 / chunks, loads = kBlock / rows_each; // 16 codes a load
    uint32_t blocks = 0;   // so far
    uint32_t segments = 0;
    bool alive = true;

    __device__ __forceinline__ void queries(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g)
    {
        constexpr uint32_t lanes = D / 8; // of a row
        const uint32_t tid = threadIdx.x - kConvert;
        alive = alive && await(s, &s.q_empty, (segments & 1u) ^ 1u);
        __syncwarp();
        const uint32_t rows = g.u.rows > kTileRows ? kUnitRows : kTileRows;
        for (uint32_t i = tid; i < rows * lanes; i += 128u) { // (whole warps: lanes is 8 or 16)
            const uint32_t r = i / lanes, chunk = i % lanes, row = g.u.row0 + r;
            const bool real = r < g.u.rows;
            uint32_t w[4] = {};
            if (real) {
                const uint64_t token = g.seq.first + row / a.group;
                const T* p = static_cast<const T*>(a.q) + token * a.q_ld + (uint64_t)(g.u.head * a.group + row % a.group) * D + chunk * 8u;
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            }
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 x = two<T>(w[k]);
                most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            __syncwarp();
#pragma unroll
            for (uint32_t d = 1; d < lanes; d <<= 1)
                most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
            // a power of two that brings the largest to 2^12; 1 where a row is nothing or infinite
            const int e = (int)(__float_as_uint(most) >> 23) - 127;
            const int up = most > 0.0f && e < 128 ? max(-100, min(100, 12 - e)) : 0;
            const float by = __uint_as_float((uint32_t)(up + 127) << 23), turned = a.scale_log2 < 0.0f ? -by : by;
            uint32_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 x = two<T>(w[k]);
                y[k] = pair_of(x.x * turned, x.y * turned);
            }
            *reinterpret_cast<uint4*>(ring.q(r / kTileRows) + tile_at(r % kTileRows, chunk)) = make_uint4(y[0], y[1], y[2], y[3]);
            if (chunk == 0) {
                const int64_t at = (int64_t)g.seq.len - g.seq.n + row / a.group;
                s.factor[r] = fmaxf(fabsf(a.scale_log2) / by, 1e-37f);
                s.hi[r] = real && at >= 0 ? (int32_t)(at + 1 < g.seq.len ? at + 1 : g.seq.len) : 0;
                s.lo[r] = a.window && at + 1 > (int64_t)a.window ? (int32_t)(at + 1 - a.window) : 0;
            }
        }
        if (tid == 0)
            s.n_mixed[segments & 1u] = 0;
        fence_proxy_async();
        __syncwarp();
        named_barrier(2, 128);
        if (tid == 0)
            mbar_arrive(&s.q_full);
        __syncwarp();
        ++segments;
    }

    // The place of this thread's token of a block (all ones: not there), and its scales.
    struct Place {
        uint64_t off;
        float key, value;
    };
    __device__ __forceinline__ Place place(const KvAttendArgs& a, const Segment& g, const int32_t* table, uint32_t block)
    {
        const uint32_t t = block * kBlock + (threadIdx.x - kConvert);
        Place p{~0ull, 0.0f, 0.0f};
        if (t < g.seq.len) {
            const uint32_t index = kv_page_of(a, t), page = (uint32_t)__ldg(table + index);
            if (page < a.c.n_pages) {
                p.off = page * a.c.page_stride + (uint64_t)g.u.head * a.c.head_stride + (uint64_t)(t - index * a.c.page_size) * a.c.token_stride;
                p.key = __ldg(a.c.k_scale + (uint64_t)page * a.c.n_heads + g.u.head);
                p.value = __ldg(a.c.v_scale + (uint64_t)page * a.c.n_heads + g.u.head);
            }
        }
        return p;
    }

    __device__ __forceinline__ void load(uint4 (&x)[loads], const void* codes, const uint64_t* off)
    {
        const uint32_t tid = threadIdx.x - kConvert, chunk = tid % chunks;
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint64_t from = off[i * rows_each + tid / chunks];
            x[i] = from != ~0ull ? __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(codes) + from + chunk * 16u)) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(const uint4 (&x)[loads], unsigned char* tile)
    {
        const uint32_t tid = threadIdx.x - kConvert, chunk = tid % chunks;
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint32_t row = i * rows_each + tid / chunks;
            const uint4 low = make_uint4(halves_of(x[i].x & 0xffffu), halves_of(x[i].x >> 16), halves_of(x[i].y & 0xffffu), halves_of(x[i].y >> 16));
            const uint4 high = make_uint4(halves_of(x[i].z & 0xffffu), halves_of(x[i].z >> 16), halves_of(x[i].w & 0xffffu), halves_of(x[i].w >> 16));
            // (the upper half of a row's lanes begin with their second half: all banks)
            const bool first = chunk < 4u;
            *reinterpret_cast<uint4*>(tile + tile_at(row, 2u * chunk + !first)) = first ? low : high;
            *reinterpret_cast<uint4*>(tile + tile_at(row, 2u * chunk + first)) = first ? high : low;
        }
    }

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g)
    {
        const uint32_t tid = threadIdx.x - kConvert, lane = tid & 31u;
        const int32_t* table = a.block_table + (uint64_t)g.sq * a.table_ld;
        float unit = 0.0f;
        Place p = place(a, g, table, g.from);
        queries(a, s, ring, g);
        s.off[blocks & 1u][tid] = p.off;
        __syncwarp();
        named_barrier(2, 128);
        uint4 k[loads], v[loads];
        load(k, a.c.k, s.off[blocks & 1u]);
        for (uint32_t b = g.from; b < g.to; ++b, ++blocks) {
            const uint32_t stage = blocks & 1u, parity = (blocks >> 1) & 1u, slot = blocks % kSlots;
            load(v, a.c.v, s.off[stage]);
            // what the softmax wants to know of the block
            float most = p.off != ~0ull ? p.value : 0.0f;
#pragma unroll
            for (uint32_t d = 16; d; d >>= 1)
                most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
            if (lane == 0)
                s.warp_most[tid / 32u] = most;
            const uint32_t missing = __ballot_sync(~0u, p.off == ~0ull && b * kBlock + tid < g.seq.len);
            alive = alive && await(s, &s.k_empty[stage], parity ^ 1u);
            __syncwarp(); // (barriers want whole warps)
            named_barrier(2, 128); // (the block before has read warp_most, and this block's are there)
            const float largest = fmaxf(fmaxf(s.warp_most[0], s.warp_most[1]), fmaxf(s.warp_most[2], s.warp_most[3]));
            const float now = fmaxf(unit, largest);
            s.scale[slot][tid] = Scale{p.key, now > 0.0f ? p.value * (kWeightUnit / now) : 0.0f};
            if (lane == 0)
                s.missing[slot][tid / 32u] = missing;
            if (tid == 0)
                s.older[slot] = now > 0.0f ? unit / now : 1.0f;
            unit = now;
            store(k, ring.k(stage));
            const bool more = b + 1u < g.to;
            if (more) {
                p = place(a, g, table, b + 1u);
                s.off[stage ^ 1u][tid] = p.off;
            } else if (tid == 0) {
                s.unit[(segments - 1u) & 1u] = unit;
            }
            fence_proxy_async();
            __syncwarp();
            named_barrier(2, 128);
            if (tid == 0)
                mbar_arrive(&s.k_full[stage]);
            __syncwarp();
            if (more)
                load(k, a.c.k, s.off[stage ^ 1u]);
            if (b * kBlock < g.see_from || (b + 1u) * kBlock > g.see_to) { // some rows see what others do not
                uint32_t bad[loads], any = 0;
#pragma unroll
                for (uint32_t i = 0; i < loads; ++i) {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                    bad[i] = 0;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        bad[i] |= __vcmpeq4(w[j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    any |= bad[i];
                }
                const uint32_t which = s.n_mixed[(segments - 1u) & 1u];
                uint32_t* at = s.mixed[(segments - 1u) & 1u][which < kMixed ? which : kMixed - 1u];
                __syncwarp();
                named_barrier(2, 128);
                if (tid < 5u)
                    at[tid] = tid ? 0u : b;
                if (tid == 0)
                    s.n_mixed[(segments - 1u) & 1u] = which < kMixed ? which + 1u : kMixed;
                __syncwarp();
                named_barrier(2, 128);
                if (any)
#pragma unroll
                    for (uint32_t i = 0; i < loads; ++i)
                        if (bad[i]) {
                            const uint32_t row = i * rows_each + tid / chunks;
                            atomicOr(at + 1u + row / 32u, 1u << (row & 31u));
                            v[i].x &= ~__vcmpeq4(v[i].x & 0x7f7f7f7fu, 0x7f7f7f7fu);
                            v[i].y &= ~__vcmpeq4(v[i].y & 0x7f7f7f7fu, 0x7f7f7f7fu);
                            v[i].z &= ~__vcmpeq4(v[i].z & 0x7f7f7f7fu, 0x7f7f7f7fu);
                            v[i].w &= ~__vcmpeq4(v[i].w & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        }
            }
            alive = alive && await(s, &s.v_empty[stage], parity ^ 1u);
            __syncwarp();
            store(v, ring.v(stage));
            fence_proxy_async();
            __syncwarp();
            named_barrier(2, 128);
            if (tid == 0)
                mbar_arrive(&s.v_full[stage]);
            __syncwarp();
        }
    }
};

// The thread that issues products.
template <uint32_t D>
struct Issuer {
    uint32_t blocks = 0, segments = 0, weights[2] = {0, 0};
    bool alive = true;

    __device__ __forceinline__ void scores(Shared& s, const Ring<D>& ring, uint32_t t, uint32_t stage)
    {
        const uint32_t desc = mma_f16_desc(false, kBlock);
#pragma unroll
        for (uint32_t k = 0; k < D / 16; ++k) {
            const uint32_t at = (k / 4u) * 16384u + (k % 4u) * 32u;
            mma_f16(s.tmem + t * 128u, smem_tile_desc(ring.q(t) + at), smem_tile_desc(ring.k(stage) + at), desc, k != 0);
        }
        mma_commit(&s.s_full[t]);
    }

    __device__ __forceinline__ void run(Shared& s, const Ring<D>& ring, const Segment& g)
    {
        const uint32_t n = g.to - g.from, tiles = g.u.rows > kTileRows ? 2u : 1u;
        const uint32_t desc = mma_f16_desc(false, D) | (1u << 16); // B is MN-major
        alive = alive && await(s, &s.q_full, segments & 1u);
        ++segments;
        alive = alive && await(s, &s.k_full[blocks & 1u], (blocks >> 1) & 1u);
        if (!alive)
            return;
        tc_fence_after();
        for (uint32_t t = 0; t < tiles; ++t)
            scores(s, ring, t, blocks & 1u);
        mma_commit(&s.k_empty[blocks & 1u]);
        if (n == 1u)
            mma_commit(&s.q_empty);
        for (uint32_t j = 0; j < n; ++j, ++blocks) {
            const uint32_t stage = blocks & 1u, parity = (blocks >> 1) & 1u, next = blocks + 1u;
            for (uint32_t t = 0; t < tiles; ++t) {
                if (t == 0 && !(alive = await(s, &s.v_full[stage], parity)))
                    return;
                if (!(alive = await(s, &s.p_full[t], weights[t] & 1u)))
                    return;
                ++weights[t];
                tc_fence_after();
                const uint64_t b = smem_rows_desc(ring.v(stage), 16384u);
#pragma unroll
                for (uint32_t k = 0; k < kBlock / 16; ++k)
                    mma_weights(s.tmem + 256u + t * 128u, s.tmem + t * 128u + k * 8u, b + k * (2048u >> 4), desc, j || k);
                if (j + 1u < n) {
                    if (t == 0 && !(alive = await(s, &s.k_full[next & 1u], (next >> 1) & 1u)))
                        return;
                    tc_fence_after();
                    scores(s, ring, t, next & 1u);
                } else {
                    mma_commit(&s.o_full[t]);
                }
            }
            mma_commit(&s.v_empty[stage]);
            if (j + 1u < n) {
                mma_commit(&s.k_empty[next & 1u]);
                if (j + 2u == n)
                    mma_commit(&s.q_empty);
            }
        }
    }
};

// Those that turn scores into weights: a row each.
template <typename T, uint32_t D>
struct Softmax {
    uint32_t blocks = 0, segments = 0, seen = 0, outputs = 0; // blocks so far of all segments, and of this tile's
    bool alive = true;

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Segment& g, float* part)
    {
        const uint32_t t = threadIdx.x / kTileRows, row = threadIdx.x, quarter = threadIdx.x / 32u % 4u;
        const uint32_t n = g.to - g.from, which = segments & 1u;
        alive = alive && await(s, &s.q_full, segments & 1u);
        ++segments;
        const float f = s.factor[row];
        const int32_t lo = s.lo[row], hi = s.hi[row];
        mbar_arrive(&s.q_empty);
        const uint32_t first = blocks;
        blocks += n;
        if (t && g.u.rows <= kTileRows)
            return;
        const uint32_t lanes = (quarter * 32u) << 16, scores = s.tmem + lanes + t * 128u, out = s.tmem + lanes + 256u + t * 128u;
        float ref = -INFINITY, l = 0.0f;
        for (uint32_t j = 0; j < n; ++j, ++seen) {
            const uint32_t slot = (first + j) % kSlots, begin = (g.from + j) * kBlock;
            alive = alive && await(s, &s.s_full[t], seen & 1u);
            __syncwarp();
            if (__any_sync(~0u, !alive)) { // (others of the CTA wait for nothing of this warp any more either)
                alive = false;
                return;
            }
            tc_fence_after();
            float x[kBlock];
#pragma unroll
            for (uint32_t i = 0; i < kBlock; i += 32)
                tmem_read32(x + i, scores + i);
            const float4* scale = reinterpret_cast<const float4*>(s.scale[slot]);
#pragma unroll
            for (uint32_t i = 0; i < kBlock; i += 2) {
                const float4 c = scale[i / 2];
                const float2 y = mul2(make_float2(x[i], x[i + 1]), make_float2(c.x, c.z));
                x[i] = y.x;
                x[i + 1] = y.y;
            }
            const uint32_t gone = s.missing[slot][0] | s.missing[slot][1] | s.missing[slot][2] | s.missing[slot][3];
            if (__any_sync(~0u, gone || lo > (int32_t)begin || hi < (int32_t)(begin + kBlock))) {
                const int32_t low = lo - (int32_t)begin, high = hi - (int32_t)begin;
                const uint32_t m[4] = {s.missing[slot][0], s.missing[slot][1], s.missing[slot][2], s.missing[slot][3]};
#pragma unroll
                for (int32_t i = 0; i < (int32_t)kBlock; ++i)
                    if (i < low || i >= high || ((m[i / 32] >> (i % 32)) & 1u))
                        x[i] = -INFINITY;
            }
            float most = x[0];
#pragma unroll
            for (uint32_t i = 1; i < kBlock; ++i)
                most = fmaxf(most, x[i]);
            most *= f;
            const float older = s.older[slot];
            float by = older;
            if (most > ref + 8.0f || ref == -INFINITY) { // (-inf: nothing seen yet; its outputs and sum are zeros)
                const float to = most > ref ? most : ref;
                by = ref == -INFINITY ? (to == -INFINITY ? older : 0.0f) : older * ex2_approx(ref - to);
                l *= ref == -INFINITY ? 1.0f : ex2_approx(ref - to);
                ref = to;
            }
            __syncwarp();
            if (j && __any_sync(~0u, by != 1.0f)) {
#pragma unroll 1
                for (uint32_t i = 0; i < D; i += 32) {
                    float y[32];
                    tmem_read32(y, out + i);
                    uint32_t z[32];
#pragma unroll
                    for (uint32_t k = 0; k < 32; ++k)
                        z[k] = __float_as_uint(y[k] * by);
                    tmem_write32(out + i, z);
                }
            }
            const float from = ref == -INFINITY ? 0.0f : ref;
            const float2 f2 = make_float2(f, f), minus = make_float2(-from, -from);
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (uint32_t i = 0; i < kBlock; i += 64) {
                uint32_t w[32];
#pragma unroll
                for (uint32_t k = 0; k < 64; k += 2) {
                    const float4 c = scale[(i + k) / 2];
                    const float2 d = fma2(make_float2(x[i + k], x[i + k + 1]), f2, minus);
                    const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y));
                    sum.x += p.x;
                    sum.y += p.y;
                    const float2 y = mul2(p, make_float2(c.y, c.w));
                    w[k / 2] = pair_of(y.x, y.y);
                }
                tmem_write32(scores + i / 2, w);
            }
            l += sum.x + sum.y;
            __syncwarp();
            tmem_written();
            tc_fence_before();
            mbar_arrive(&s.p_full[t]);
            __syncwarp();
        }
        alive = alive && await(s, &s.o_full[t], outputs & 1u);
        ++outputs;
        __syncwarp();
        if (__any_sync(~0u, !alive)) {
            alive = false;
            return;
        }
        tc_fence_after();
        for (uint32_t i = 0; i < s.n_mixed[which]; ++i) { // values that are NaN, of blocks that not all rows see
            const uint32_t* b = s.mixed[which][i];
            for (uint32_t k = 0; k < kBlock; ++k) {
                const int32_t key = (int32_t)(b[0] * kBlock + k);
                if (!b[1] && !b[2] && !b[3] && !b[4])
                    break;
                if (((b[1 + k / 32u] >> (k & 31u)) & 1u) && key >= lo && key < hi)
                    l = __int_as_float(0x7fc00000);
            }
        }
        __syncwarp();
        const bool real = row < g.u.rows;
        const float worth = s.unit[which] / kWeightUnit;
        const uint32_t r = g.u.row0 + row;
        T* to = static_cast<T*>(a.out) + (g.seq.first + r / a.group) * a.out_ld + (uint64_t)(g.u.head * a.group + r % a.group) * D;
        const float by = part ? worth : l == 0.0f ? 0.0f : worth / l;
#pragma unroll 1
        for (uint32_t i = 0; i < D; i += 32) {
            float y[32];
            tmem_read32(y, out + i);
            if (real && part) {
#pragma unroll
                for (uint32_t k = 0; k < 32; k += 4)
                    *reinterpret_cast<float4*>(part + row * D + i + k) = make_float4(y[k] * by, y[k + 1] * by, y[k + 2] * by, y[k + 3] * by);
            } else if (real) {
#pragma unroll
                for (uint32_t k = 0; k < 32; k += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        if constexpr (std::is_same<T, __half>::value) {
                            w[m] = pair_of(y[k + 2 * m] * by, y[k + 2 * m + 1] * by);
                        } else {
                            const __nv_bfloat162 z = __floats2bfloat162_rn(y[k + 2 * m] * by, y[k + 2 * m + 1] * by);
                            w[m] = *reinterpret_cast<const uint32_t*>(&z);
                        }
                    }
                    *reinterpret_cast<uint4*>(to + i + k) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            __syncwarp();
        }
        tc_fence_before();
        if (real && part) {
            part[kUnitRows * D + row] = ref;
            part[kUnitRows * (D + 1u) + row] = l;
        }
    }
};

template <typename T, uint32_t D>
__global__ void __launch_bounds__(kThreads, 1) kv_prompt_kernel(const KvAttendArgs a)
{
    extern __shared__ unsigned char raw[];
    __shared__ Shared s;
    Ring<D> ring;
    ring.base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    const uint32_t tid = threadIdx.x, warp = tid / 32u;
    if (tid == 0) {
        mbar_init(&s.q_full, 1);
        mbar_init(&s.q_empty, 1u + 2u * kTileRows);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&s.k_full[i], 1);
            mbar_init(&s.k_empty[i], 1);
            mbar_init(&s.v_full[i], 1);
            mbar_init(&s.v_empty[i], 1);
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], kTileRows);
            mbar_init(&s.o_full[i], 1);
        }
        s.failed = 0;
        fence_barrier_init();
    }
    if (warp == kIssue / 32u)
        tmem_alloc_all(&s.tmem);
    griddep_launch_dependents();
    griddep_wait();
    uint64_t begin, end, total;
    uint32_t ctas;
    tc_fence_before();
    const KvAt found = kv_find<kThreads>(a, kUnitRows, kBlock, gridDim.x, a.blocks_least, s.find, blockIdx.x, begin, end, total, ctas);
    tc_fence_after();
    // each of them goes through the CTA's segments
    auto segments = [&](auto&& role) {
        uint64_t at = begin, off = found.off;
        for (uint32_t sq = found.seq; at < end && sq < a.n_seq; ++sq, off = 0) {
            Segment g;
            g.sq = sq;
            g.seq = kv_seq(a, sq);
            const uint32_t per_head = kv_seq_blocks(a, g.seq, kUnitRows, kBlock);
            while (at < end && off < (uint64_t)per_head * a.c.n_heads) {
                g.u = kv_unit(a, g.seq, per_head, off, kUnitRows, kBlock);
                g.from = g.u.blocks.from + g.u.skip;
                g.to = end - at < g.u.blocks.to - g.from ? g.from + (uint32_t)(end - at) : g.u.blocks.to;
                const int64_t back = (int64_t)g.seq.len - g.seq.n, top = back + g.u.row0 / a.group + 1, last = back + (g.u.row0 + g.u.rows - 1u) / a.group + 1;
                g.see_to = top < 0 ? 0u : top < g.seq.len ? (uint32_t)top : g.seq.len;
                g.see_from = a.window && last > (int64_t)a.window ? (uint32_t)(last - a.window) : 0u;
                const bool whole = g.u.skip == 0 && g.to == g.u.blocks.to;
                float* part = whole ? nullptr : a.parts + (uint64_t)(2u * blockIdx.x + (at != begin)) * (kUnitRows * (D + 2u));
                role(g, part);
                at += g.to - g.from;
                off += g.to - g.from;
            }
        }
    };
    // 128 registers a thread at launch: 256 x 184 + 128 x 104 + 128 x 40 = 512 x 128
    if (blockIdx.x < ctas) {
        if (tid < kConvert) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
            Softmax<T, D> x;
            segments([&](const Segment& g, float* part) { x.run(a, s, g, part); });
        } else if (tid < kIssue) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
            Converter<T, D> x;
            segments([&](const Segment& g, float*) { x.run(a, s, ring, g); });
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
            if (tid == kIssue) {
                Issuer<D> x;
                segments([&](const Segment& g, float*) {
                    if (x.alive)
                        x.run(s, ring, g);
                });
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (s.failed) { // never seen: products in flight end within this, and the rows say what happened
        for (int i = 0; i < 2000; ++i)
            __nanosleep(1000);
        for (uint64_t i = tid; i < (uint64_t)a.n_tokens * a.group * a.c.n_heads * D; i += kThreads) {
            const uint64_t width = (uint64_t)a.group * a.c.n_heads * D;
            static_cast<uint16_t*>(a.out)[i / width * a.out_ld + i % width] = 0x7fffu;
        }
        __syncthreads();
    }
    if (warp == kIssue / 32u)
        tmem_free_all(s.tmem);
}

template <typename T, uint32_t D>
cudaError_t launch(const KvAttendArgs& a, cudaStream_t stream)
{
    constexpr uint32_t smem = 6u * Ring<D>::tile_bytes + 1024u;
    static const bool split_fits = [] { // the registers that the warps share out among themselves are those of the launch
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, kv_prompt_kernel<T, D>) == cudaSuccess && f.numRegs == 128;
    }();
    if (!split_fits)
        return cudaErrorInvalidKernelImage;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = set_once(done, kv_prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess)
        return e;
    kv_prompt_kernel<T, D><<<kPromptCtas, kThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

} // namespace

cudaError_t launch_kv_prompt(const KvAttendArgs& a, int type, cudaStream_t stream)
{
    if (type == MK_BF16)
        return a.c.dim == 128u ? launch<__nv_bfloat16, 128>(a, stream) : launch<__nv_bfloat16, 64>(a, stream);
    return a.c.dim == 128u ? launch<__half, 128>(a, stream) : launch<__half, 64>(a, stream);
}

} // namespace mk
