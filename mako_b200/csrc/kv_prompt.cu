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
constexpr uint32_t kThreads = 416; // of 128 registers each
constexpr uint32_t kConvert = 256, kIssue = 384; // first thread of those that convert, and of the warp that issues
constexpr uint32_t kSlots = 4;                   // of what softmax reads beside the scores
constexpr float kWeightUnit = 128.0f;
constexpr uint32_t kMixed = 8; // blocks of a segment that some rows see and others do not: at most 3 at either end

struct Shared {
    uint64_t find[40];
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int failed;
    alignas(16) float key[kSlots][kBlock], value[kSlots][kBlock]; // scales; values' over the largest so far, times kWeightUnit
    alignas(16) uint32_t missing[kSlots][4]; // tokens whose page is not there
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
__device__ __forceinline__ void tmem_read64(float* x, uint32_t at)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, "
        "%56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : MK_R8(x, 0), MK_R8(x, 8), MK_R8(x, 16), MK_R8(x, 24), MK_R8(x, 32), MK_R8(x, 40), MK_R8(x, 48), MK_R8(x, 56)
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
__device__ __forceinline__ void tmem_write16(uint32_t at, const uint32_t* x)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::MK_W8(x, 0),
        MK_W8(x, 8), "r"(at)
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

struct Segment : KvSegment {
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
    // a load is 16 codes: of 32 rows, 64 columns. (Eight lanes have two rows' quarters: their stores are in different banks.)
    static constexpr uint32_t halves = D / 64, loads = kBlock / 32 * halves;
    static __device__ __forceinline__ uint32_t row_of(uint32_t i) { return i / halves * 32u + (threadIdx.x - kConvert) / 4u; }
    static __device__ __forceinline__ uint32_t chunk_of(uint32_t i) { return i % halves * 4u + (threadIdx.x & 3u); }
    uint32_t blocks = 0;   // so far
    uint32_t segments = 0;
    bool alive = true;

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
                p.off = page * a.c.page_stride + (uint64_t)g.head * a.c.head_stride + (uint64_t)(t - index * a.c.page_size) * a.c.token_stride;
                p.key = __ldg(a.c.k_scale + (uint64_t)page * a.c.n_heads + g.head);
                p.value = __ldg(a.c.v_scale + (uint64_t)page * a.c.n_heads + g.head);
            }
        }
        return p;
    }

    __device__ __forceinline__ void load(uint4 (&x)[loads], const void* codes, const uint64_t* off)
    {
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint64_t from = off[row_of(i)];
            x[i] = from != ~0ull ? __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(codes) + from + chunk_of(i) * 16u)) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(const uint4 (&x)[loads], unsigned char* tile)
    {
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint2 y0 = halves_of4(x[i].x), y1 = halves_of4(x[i].y), y2 = halves_of4(x[i].z), y3 = halves_of4(x[i].w);
            *reinterpret_cast<uint4*>(tile + tile_at(row_of(i), 2u * chunk_of(i))) = make_uint4(y0.x, y0.y, y1.x, y1.y);
            *reinterpret_cast<uint4*>(tile + tile_at(row_of(i), 2u * chunk_of(i) + 1u)) = make_uint4(y2.x, y2.y, y3.x, y3.y);
        }
    }

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g)
    {
        const uint32_t tid = threadIdx.x - kConvert, lane = tid & 31u;
        const int32_t* table = a.block_table + (uint64_t)g.sq * a.table_ld;
        float unit = 0.0f;
        Place p = place(a, g, table, g.from);
        if (tid == 0)
            s.n_mixed[segments & 1u] = 0; // (that of the segment before the last one has been read: its successor's softmax has begun)
        ++segments;
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
            s.key[slot][tid] = p.key;
            s.value[slot][tid] = now > 0.0f ? p.value * (kWeightUnit / now) : 0.0f;
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
                            const uint32_t row = row_of(i);
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
        const uint32_t n = g.to - g.from, tiles = g.rows > kTileRows ? 2u : 1u;
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

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g, float* part)
    {
        const uint32_t t = threadIdx.x / kTileRows, row = threadIdx.x, quarter = threadIdx.x / 32u % 4u;
        const uint32_t n = g.to - g.from, which = segments & 1u;
        // the row's queries, times a power of two that brings the largest to 2^12 (1 where a row is nothing or infinite)
        const uint32_t unit_row = g.row0 + row, token = kv_token_of(a, unit_row), head = g.head * a.group + (unit_row - token * a.group);
        const bool real = row < g.rows;
        float f;
        {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (g.seq.first + token) * a.q_ld + (uint64_t)head * D);
            uint4 q[D / 8];
#pragma unroll
            for (uint32_t i = 0; i < D / 8; ++i)
                q[i] = real ? __ldg(p + i) : make_uint4(0, 0, 0, 0);
            float top = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < D / 8; ++i) {
                const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 x = two<T>(w[k]);
                    top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                }
            }
            const int e = (int)(__float_as_uint(top) >> 23) - 127;
            const int up = top > 0.0f && e < 128 ? max(-100, min(100, 12 - e)) : 0;
            const float by = __uint_as_float((uint32_t)(up + 127) << 23), turned = a.scale_log2 < 0.0f ? -by : by;
            f = fmaxf(fabsf(a.scale_log2) / by, 1e-37f); // (not 0: a key that the row does not see has -inf times this)
            alive = alive && await(s, &s.q_empty, (segments & 1u) ^ 1u);
            ++segments;
            unsigned char* tile = ring.q(t);
#pragma unroll
            for (uint32_t i = 0; i < D / 8; ++i) {
                const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
                uint32_t y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 x = two<T>(w[k]);
                    y[k] = pair_of(x.x * turned, x.y * turned);
                }
                *reinterpret_cast<uint4*>(tile + tile_at(row % kTileRows, i)) = make_uint4(y[0], y[1], y[2], y[3]);
            }
            fence_proxy_async();
            mbar_arrive(&s.q_full);
        }
        const int32_t at = (int32_t)g.seq.len - (int32_t)g.seq.n + (int32_t)token + 1; // behind its position
        const int32_t hi = real && at > 0 ? at : 0, lo = a.window && at > (int32_t)a.window ? at - (int32_t)a.window : 0;
        const uint32_t first = blocks;
        blocks += n;
        __syncwarp();
        if (t && g.rows <= kTileRows)
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
            const float4 *key = reinterpret_cast<const float4*>(s.key[slot]), *value = reinterpret_cast<const float4*>(s.value[slot]);
            const uint4 gone = *reinterpret_cast<const uint4*>(s.missing[slot]);
            const int32_t low = lo - (int32_t)begin, high = hi - (int32_t)begin;
            const bool some = __any_sync(~0u, (gone.x | gone.y | gone.z | gone.w) != 0 || low > 0 || high < (int32_t)kBlock);
            // Half of a row's scores, times the keys' scales; -inf where it does not see the key. (A thread has registers for half of them: the
            // second half is read twice, for the largest and once the first half's weights are made.)
            auto read = [&](float (&x)[64], uint32_t half) {
                tmem_read64(x, scores + 64u * half);
#pragma unroll
                for (uint32_t i = 0; i < 64; i += 4) {
                    const float4 c = key[16u * half + i / 4];
                    const float2 y = mul2(make_float2(x[i], x[i + 1]), make_float2(c.x, c.y)), z = mul2(make_float2(x[i + 2], x[i + 3]), make_float2(c.z, c.w));
                    x[i] = y.x, x[i + 1] = y.y, x[i + 2] = z.x, x[i + 3] = z.y;
                }
                if (some) {
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const int32_t from = low - 64 * (int32_t)half - 32 * (int32_t)i, to = high - 64 * (int32_t)half - 32 * (int32_t)i;
                        // the places [from, to) of 32
                        const uint32_t behind = to <= 0 ? 0u : to >= 32 ? ~0u : (1u << to) - 1u;
                        const uint32_t before = from <= 0 ? 0u : from >= 32 ? ~0u : (1u << from) - 1u;
                        const uint32_t sees = behind & ~before & ~(half ? (i ? gone.w : gone.z) : (i ? gone.y : gone.x));
#pragma unroll
                        for (uint32_t k = 0; k < 32; ++k)
                            x[32 * i + k] = (sees >> k) & 1u ? x[32 * i + k] : -INFINITY;
                    }
                }
            };
            float x[64], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int half = 1; half >= 0; --half) {
                read(x, half);
#pragma unroll
                for (uint32_t i = 0; i < 64; i += 8)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        tops[k] = fmaxf(tops[k], fmaxf(x[i + k], x[i + k + 4]));
            }
            const float most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * f;
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
            float2 sum = make_float2(0.0f, 0.0f), more = sum;
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                if (half)
                    read(x, 1u);
#pragma unroll
                for (uint32_t i0 = 0; i0 < 64; i0 += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (uint32_t i = i0; i < i0 + 32; i += 4) {
                        const float4 c = value[16u * half + i / 4];
                        const float2 d = fma2(make_float2(x[i], x[i + 1]), f2, minus), e = fma2(make_float2(x[i + 2], x[i + 3]), f2, minus);
                        const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y)), q = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                        sum = add2(sum, p);
                        more = add2(more, q);
                        const float2 y = mul2(p, make_float2(c.x, c.y)), z = mul2(q, make_float2(c.z, c.w));
                        w[(i - i0) / 2] = pair_of(y.x, y.y);
                        w[(i - i0) / 2 + 1] = pair_of(z.x, z.y);
                    }
                    tmem_write16(scores + 32u * half + i0 / 2, w); // (over the first half's scores, which have been read)
                }
            }
            l += (sum.x + sum.y) + (more.x + more.y);
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
        const float worth = s.unit[which] / kWeightUnit;
        T* to = static_cast<T*>(a.out) + (g.seq.first + token) * a.out_ld + (uint64_t)head * D;
        const float by = part ? worth : l == 0.0f ? 0.0f : worth / l;
#pragma unroll 1
        for (uint32_t i = 0; i < D; i += 32) {
            float y[32];
            tmem_read32(y, out + i);
            if (real && part) {
#pragma unroll
                for (uint32_t k = 0; k < 32; ++k)
                    part[(i + k) * kUnitRows + row] = y[k] * by; // (by column: lanes are rows)
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
        mbar_init(&s.q_full, kUnitRows);
        mbar_init(&s.q_empty, 1);
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
    tc_fence_before();
    const KvWalk found = kv_find<kThreads>(a, kUnitRows, kBlock, gridDim.x, s.find, blockIdx.x);
    tc_fence_after();
    // each of them goes through the CTA's segments
    auto segments = [&](auto&& role) {
        KvWalk walk = found;
        Segment g;
        for (bool first = true; kv_take(a, walk, g, first, kUnitRows, kBlock); first = false) {
            const int32_t back = (int32_t)g.seq.len - (int32_t)g.seq.n;
            const int32_t top = back + (int32_t)kv_token_of(a, g.row0) + 1, last = back + (int32_t)kv_token_of(a, g.row0 + g.rows - 1u) + 1;
            g.see_to = top < 0 ? 0u : (uint32_t)top;
            g.see_from = a.window && last > (int32_t)a.window ? (uint32_t)last - a.window : 0u;
            role(g, g.whole() ? nullptr : a.parts + (uint64_t)(2u * blockIdx.x + !first) * (kUnitRows * (D + 2u)));
        }
    };
    if (blockIdx.x < found.ctas) {
        if (tid < kConvert) {
            Softmax<T, D> x;
            segments([&](const Segment& g, float* part) { x.run(a, s, ring, g, part); });
        } else if (tid < kIssue) {
            Converter<T, D> x;
            segments([&](const Segment& g, float*) { x.run(a, s, ring, g); });
        } else {
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
