// Attention of many rows over a paged 8-bit cache (mk_kv_attention in include/mako_b200.h): prompts' chunks. The tensor core's work is 2048 cycles
// for a block of 128 keys past 256 rows of 128 columns, as much as its exponentials take; a block takes about 5100 (4 chunks of 2048
// tokens at the end of 8192, 32 query heads on 8: 1295 us, 743 TFLOP/s, 0.45 of the measured rate of a matrix product). What it waits for
// is the chain of a tile's turn: scores out of tensor memory, their largest, exponentials, weights back, two products and their signals, with
// the conversion beside it; shared memory is two fifths busy.
//
// A unit has 256 rows, two tiles of the MMA's M, that take turns: while one tile's scores become weights, the tensor core works for the
// other. One warp issues; eight a tile (two threads a row) turn scores into weights; four turn the cache's codes into fp16, K-major for the
// keys, the same bytes read as MN-major for the values. Scores and outputs are in tensor memory; weights take the scores' place, as the A
// operand of the second product. A sum is multiplied only where a row's maximum has grown by more than 2^8, outputs where the row's largest weight
// has (kv_unit in kv_work.cuh). Rounding is that of kv_attend.cu: queries, codes exactly, weights to fp16.
//
// What it came from: a thread a row with its 128 scores in registers 2058 us (registers are shared by 12 warps then), half of them at a time
// 1650; two threads a row did not help until a scale for each key was no longer read for each (shared memory: 52 % to 35 %; 1580); pages looked
// up two blocks ahead 1448; a block's codes read a block ahead 1361 (1358 to
// 1420 from one device to another); units of the rows' own in place of the converters' common one, which had them wait for one another, 1410 -> 1295.
// Pages that are no multiple of 16 tokens: 1654 (of 24 tokens; 1580 with the common unit).
#include "kv_cache.cuh"
#include "kv_work.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>

namespace mk {
namespace {

constexpr uint32_t kTileRows = 128, kUnitRows = 256, kBlock = 128; // rows of a tile, of a unit; keys of a block
constexpr uint32_t kThreads = 672;
constexpr uint32_t kConvert = 512, kIssue = 640; // first thread of those that convert, and of the warp that issues
constexpr uint32_t kSlots = 4;                   // of what softmax reads beside the scores
constexpr uint32_t kMixed = 8; // blocks of a segment that some rows see and others do not: at most 3 at either end
// Places for what a segment's softmax reads at its end, by the segment's number. Those that convert wait for products alone, and a segment may
// be one block long: at the end of a segment s - 1 they know that the scores of the block two before its last are done. With segments s - 3
// and s - 2 in front of it that block is of s - 3 at least, whose scores wait for all of its queries (q_full), and there every thread of the
// softmax arrives behind its segment s - 4. (With two places a short segment's outputs got the unit of the one after the next.)
constexpr uint32_t kHeld = 4;

struct Shared {
    uint64_t find[40];
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int failed;
    alignas(16) float key[kSlots][kBlock], value[kSlots][kBlock], value_log[kSlots][kBlock]; // scales; log2 of values'
    float2 log_range[kSlots][kBlock / 32]; // of 32 of them: the largest and the smallest
    alignas(16) uint32_t missing[kSlots][4]; // tokens whose page is not there
    uint32_t n_mixed[kHeld];
    uint32_t mixed[kHeld][kMixed][5];  // a block and which of its values are NaN
    uint64_t off[2][kBlock];
    float top[2][kUnitRows], most[2][kUnitRows], sum[2][kUnitRows]; // what the two threads of a row tell one another
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
    __device__ __forceinline__ uint4* wait() const { return reinterpret_cast<uint4*>(base + 6u * tile_bytes); } // a block's codes
    static constexpr uint32_t bytes = 6u * tile_bytes + kBlock * D;
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

    // The page of this thread's token of a block (all ones: not there), two blocks ahead; the token's place in it and its scales, one ahead:
    // each is there when the next one is read with it.
    __device__ __forceinline__ uint32_t look_up(const KvAttendArgs& a, const Segment& g, const int32_t* table, uint32_t block)
    {
        const uint32_t t = block * kBlock + (threadIdx.x - kConvert);
        return block < g.to && t < g.seq.keys ? (uint32_t)__ldg(table + kv_page_of(a, t)) : ~0u;
    }
    struct Place {
        uint64_t off;
        float key, value;
    };
    __device__ __forceinline__ Place place(const KvAttendArgs& a, const Segment& g, uint32_t page, uint32_t block)
    {
        Place p{~0ull, 0.0f, 0.0f};
        if (page < a.c.n_pages) {
            const uint32_t t = block * kBlock + (threadIdx.x - kConvert), in_page = t - kv_page_of(a, t) * a.c.page_size;
            p.off = page * a.c.page_stride + (uint64_t)g.head * a.c.head_stride + (uint64_t)in_page * a.c.token_stride;
            p.key = __ldg(a.c.k_scale + (uint64_t)page * a.c.n_heads + g.head);
            p.value = __ldg(a.c.v_scale + (uint64_t)page * a.c.n_heads + g.head);
        }
        return p;
    }

    // A block's values wait in registers and its keys in shared memory, each thread's own, until the block before is done with: a read that L2
    // does not answer takes 3000 cycles, as long as turning a block into fp16.
    __device__ __forceinline__ void load(uint4 (&x)[loads], const void* codes, const uint64_t* off)
    {
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint64_t from = off[row_of(i)];
            x[i] = from != ~0ull ? __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(codes) + from + chunk_of(i) * 16u)) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void copy(uint4* wait, const void* codes, const uint64_t* off)
    {
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            const uint64_t from = off[row_of(i)];
            const unsigned char* p = static_cast<const unsigned char*>(codes) + (from != ~0ull ? from + chunk_of(i) * 16u : 0ull);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(wait + i * 128u + threadIdx.x - kConvert)), "l"(p),
                         "r"(from != ~0ull ? 16u : 0u)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ void store(const uint4& x, unsigned char* tile, uint32_t i)
    {
        const uint2 y0 = halves_of4(x.x), y1 = halves_of4(x.y), y2 = halves_of4(x.z), y3 = halves_of4(x.w);
        *reinterpret_cast<uint4*>(tile + tile_at(row_of(i), 2u * chunk_of(i))) = make_uint4(y0.x, y0.y, y1.x, y1.y);
        *reinterpret_cast<uint4*>(tile + tile_at(row_of(i), 2u * chunk_of(i) + 1u)) = make_uint4(y2.x, y2.y, y3.x, y3.y);
    }
    // Takes values that are NaN out, and says whose they are.
    __device__ __forceinline__ void take_out(uint4 (&x)[loads], uint32_t* whose)
    {
#pragma unroll
        for (uint32_t i = 0; i < loads; ++i) {
            uint32_t* w[4] = {&x[i].x, &x[i].y, &x[i].z, &x[i].w};
            uint32_t bad = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t nan = __vcmpeq4(*w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                *w[k] &= ~nan;
                bad |= nan;
            }
            if (bad)
                atomicOr(whose + row_of(i) / 32u, 1u << (row_of(i) & 31u));
        }
    }

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g)
    {
        const uint32_t tid = threadIdx.x - kConvert, lane = tid & 31u, held = segments++ % kHeld;
        const int32_t* table = a.block_table + (uint64_t)g.sq * a.table_ld;
        Place p = place(a, g, look_up(a, g, table, g.from), g.from);
        uint32_t page = look_up(a, g, table, g.from + 1u);
        if (tid == 0)
            s.n_mixed[held] = 0; // (see kHeld)
        s.off[blocks & 1u][tid] = p.off;
        __syncwarp();
        named_barrier(2, 128);
        uint4* keys = ring.wait();
        uint4 v[loads];
        copy(keys, a.c.k, s.off[blocks & 1u]);
        load(v, a.c.v, s.off[blocks & 1u]);
        for (uint32_t b = g.from; b < g.to; ++b, ++blocks) {
            const uint32_t stage = blocks & 1u, parity = (blocks >> 1) & 1u, slot = blocks % kSlots;
            const bool more = b + 1u < g.to;
            const Place next = place(a, g, page, b + 1u);
            page = look_up(a, g, table, b + 2u);
            s.off[stage ^ 1u][tid] = next.off;
            // what the softmax wants to know of the block
            const uint32_t missing = __ballot_sync(~0u, p.off == ~0ull && b * kBlock + tid < g.seq.keys);
            alive = alive && await(s, &s.k_empty[stage], parity ^ 1u);
            __syncwarp(); // (barriers want whole warps)
            s.key[slot][tid] = p.key;
            s.value[slot][tid] = p.value;
            s.value_log[slot][tid] = __log2f(p.value);
            if (a.c.page_size % 16u) { // (else 16 have one. Scales are not below 0: as bits they are in the order of numbers)
                const uint32_t most = __reduce_max_sync(~0u, p.off != ~0ull ? __float_as_uint(p.value) : 0u);
                const uint32_t least = __reduce_min_sync(~0u, p.off != ~0ull ? __float_as_uint(p.value) : 0x7f800000u);
                if (lane == 0)
                    s.log_range[slot][tid / 32u] = make_float2(__log2f(__uint_as_float(most)), __log2f(__uint_as_float(least)));
            }
            if (lane == 0)
                s.missing[slot][tid / 32u] = missing;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
            for (uint32_t i = 0; i < loads; ++i)
                store(keys[i * 128u + tid], ring.k(stage), i);
            p = next;
            fence_proxy_async();
            __syncwarp();
            named_barrier(2, 128);
            if (tid == 0)
                mbar_arrive(&s.k_full[stage]);
            __syncwarp();
            if (more)
                copy(keys, a.c.k, s.off[stage ^ 1u]);
            if (b * kBlock < g.see_from || (b + 1u) * kBlock > g.see_to) { // some rows see what others do not
                const uint32_t which = s.n_mixed[held];
                uint32_t* at = s.mixed[held][which < kMixed ? which : kMixed - 1u];
                __syncwarp();
                named_barrier(2, 128);
                if (tid < 5u)
                    at[tid] = tid ? 0u : b;
                if (tid == 0)
                    s.n_mixed[held] = which < kMixed ? which + 1u : kMixed;
                __syncwarp();
                named_barrier(2, 128);
                take_out(v, at + 1);
                __syncwarp();
            }
            alive = alive && await(s, &s.v_empty[stage], parity ^ 1u);
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i < loads; ++i)
                store(v[i], ring.v(stage), i);
            if (more)
                load(v, a.c.v, s.off[stage ^ 1u]);
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
                    mma_weights(s.tmem + 256u + t * 128u, s.tmem + t * 128u + k / 4u * 64u + k % 4u * 8u, b + k * (2048u >> 4), desc, j || k);
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

// Those that turn scores into weights: two threads a row, of half of a block's keys, and of a row's columns, each. They are in different
// warps (a warp has access to 32 rows of tensor memory), so that four warps of each scheduler have scores under way. Group: keys, side by
// side, that have one scale: 16 where pages are a multiple of that, else 1. Reading a scale for each key from shared memory takes as much of
// it as the products' operands do.
template <typename T, uint32_t D, uint32_t Group>
struct Softmax {
    uint32_t blocks = 0, segments = 0, seen = 0, outputs = 0; // blocks so far of all segments, and of this tile's
    bool alive = true;

    __device__ __forceinline__ void run(const KvAttendArgs& a, Shared& s, const Ring<D>& ring, const Segment& g, float* part)
    {
        constexpr uint32_t columns = D / 2;
        const uint32_t warp = threadIdx.x / 32u, t = warp / 8u, half = warp / 4u % 2u, quarter = warp % 4u;
        const uint32_t row = t * kTileRows + quarter * 32u + (threadIdx.x & 31u), pair = 3u + t * 4u + quarter;
        const uint32_t n = g.to - g.from, which = segments % kHeld;
        // the row's queries, times a power of two that brings the largest to 2^12 (1 where a row is nothing or infinite)
        const uint32_t unit_row = g.row0 + row, token = kv_token_of(a, unit_row), head = g.head * a.group + (unit_row - token * a.group);
        const bool real = row < g.rows;
        float f;
        {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (g.seq.first + token) * a.q_ld + (uint64_t)head * D + half * columns);
            uint4 q[columns / 8];
#pragma unroll
            for (uint32_t i = 0; i < columns / 8; ++i)
                q[i] = real ? __ldg(p + i) : make_uint4(0, 0, 0, 0);
            float top = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < columns / 8; ++i) {
                const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 x = two<T>(w[k]);
                    top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                }
            }
            s.top[half][row] = top;
            __syncwarp();
            named_barrier(pair, 64);
            top = fmaxf(top, s.top[half ^ 1u][row]);
            const int e = (int)(__float_as_uint(top) >> 23) - 127;
            const int up = top > 0.0f && e < 128 ? min(100, 12 - e) : 0;
            const float by = __uint_as_float((uint32_t)(up + 127) << 23), turned = a.scale_log2 < 0.0f ? -by : by;
            f = fmaxf(fabsf(a.scale_log2) / by, 1e-37f); // (not 0: a key that the row does not see has -inf times this)
            alive = alive && await(s, &s.q_empty, (segments & 1u) ^ 1u);
            ++segments;
            unsigned char* tile = ring.q(t);
#pragma unroll
            for (uint32_t i = 0; i < columns / 8; ++i) {
                const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
                uint32_t y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 x = two<T>(w[k]);
                    y[k] = pair_of(x.x * turned, x.y * turned);
                }
                *reinterpret_cast<uint4*>(tile + tile_at(row % kTileRows, half * (columns / 8) + i)) = make_uint4(y[0], y[1], y[2], y[3]);
            }
            fence_proxy_async();
            mbar_arrive(&s.q_full);
        }
        const int32_t at = (int32_t)g.seq.len - (int32_t)g.seq.n + (int32_t)token + 1; // behind its position
        const int32_t hi = real && at > 0 ? min(at, (int32_t)g.seq.keys) : 0, lo = a.window && at > (int32_t)a.window ? at - (int32_t)a.window : 0;
        const uint32_t first = blocks;
        blocks += n;
        __syncwarp();
        if (t && g.rows <= kTileRows)
            return;
        const uint32_t lanes = (quarter * 32u) << 16, scores = s.tmem + lanes + t * 128u + half * 64u, out = s.tmem + lanes + 256u + t * 128u + half * columns;
        float ref = -INFINITY, unit = INFINITY, l = 0.0f;
        for (uint32_t j = 0; j < n; ++j, ++seen) {
            const uint32_t slot = (first + j) % kSlots, begin = (g.from + j) * kBlock;
            alive = alive && await(s, &s.s_full[t], seen & 1u);
            __syncwarp(); // (a warp that gave up goes on: its row's other thread meets it at barriers)
            tc_fence_after();
            const float *key = s.key[slot] + 64u * half, *value = s.value[slot] + 64u * half, *value_log = s.value_log[slot] + 64u * half;
            const uint2 gone = *reinterpret_cast<const uint2*>(&s.missing[slot][2u * half]);
            const int32_t low = lo - (int32_t)(begin + 64u * half), high = hi - (int32_t)(begin + 64u * half);
            const bool some = __any_sync(~0u, (gone.x | gone.y) != 0 || low > 0 || high < 64);
            // 32 of the row's scores, times the keys' scales where those are not taken in with f; -inf where it does not see the key. (They are
            // read twice, for the largest first: registers for them are not worth having half as many warps.)
            auto read = [&](float (&x)[32], uint32_t i) {
                tmem_read32(x, scores + 32u * i);
                if constexpr (Group == 1) {
#pragma unroll
                    for (uint32_t k = 0; k < 32; k += 4) {
                        const float4 c = reinterpret_cast<const float4*>(key)[8u * i + k / 4];
                        const float2 y = mul2(make_float2(x[k], x[k + 1]), make_float2(c.x, c.y)), z = mul2(make_float2(x[k + 2], x[k + 3]), make_float2(c.z, c.w));
                        x[k] = y.x, x[k + 1] = y.y, x[k + 2] = z.x, x[k + 3] = z.y;
                    }
                }
                if (some) {
                    const int32_t from = low - 32 * (int32_t)i, to = high - 32 * (int32_t)i;
                    // the places [from, to) of 32
                    const uint32_t behind = to <= 0 ? 0u : to >= 32 ? ~0u : (1u << to) - 1u, before = from <= 0 ? 0u : from >= 32 ? ~0u : (1u << from) - 1u;
                    const uint32_t sees = behind & ~before & ~(i ? gone.y : gone.x);
#pragma unroll
                    for (uint32_t k = 0; k < 32; ++k)
                        x[k] = (sees >> k) & 1u ? x[k] : -INFINITY;
                }
            };
            // what makes exponents of 16 scores (not 0, as f)
            auto factor = [&](uint32_t i) { return Group == 1 ? f : fmaxf(f * key[i], 1e-37f); };
            float most = -INFINITY, peak = -INFINITY; // log2 of the largest p and of the largest weight
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                float x[32];
                read(x, i);
#pragma unroll
                for (uint32_t k = 0; k < 32; k += 16) {
                    float tops[4];
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m)
                        tops[m] = fmaxf(fmaxf(x[k + m], x[k + m + 4]), fmaxf(x[k + m + 8], x[k + m + 12]));
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * factor(32u * i + k);
                    most = fmaxf(most, top);
                    peak = fmaxf(peak, top + (Group == 1 ? s.log_range[slot][2u * half + i].x : value_log[32u * i + k]));
                }
            }
            if constexpr (Group == 1) { // where scales are far from one another and the unit may have to grow: each by itself
                const float2 first = s.log_range[slot][2u * half], second = s.log_range[slot][2u * half + 1u];
                const bool far = !(first.x - first.y <= kHighSlack) || !(second.x - second.y <= kHighSlack); // (in all lanes)
                if (far && __any_sync(~0u, peak > unit + 15.0f || unit == INFINITY)) {
                    peak = -INFINITY;
#pragma unroll 1
                    for (uint32_t i = 0; i < 2; ++i) {
                        float x[32];
                        read(x, i);
#pragma unroll
                        for (uint32_t k = 0; k < 32; k += 2) {
                            const float2 c = reinterpret_cast<const float2*>(value_log)[16u * i + k / 2];
                            const float2 y = fma2(make_float2(x[k], x[k + 1]), make_float2(f, f), c);
                            peak = fmaxf(peak, fmaxf(y.x, y.y));
                        }
                    }
                }
            }
            s.most[half][row] = most;
            s.top[half][row] = peak;
            __syncwarp();
            named_barrier(pair, 64);
            most = fmaxf(most, s.most[half ^ 1u][row]);
            peak = fmaxf(peak, s.top[half ^ 1u][row]);
            if (most > ref + 8.0f || ref == -INFINITY) { // (-inf: nothing seen yet; its outputs and sum are zeros)
                const float to = most > ref ? most : ref;
                l *= ref == -INFINITY ? 1.0f : ex2_approx(ref - to);
                ref = to;
            }
            const float now = kv_unit(unit, peak, ref), by = now == unit ? 1.0f : kv_worth(unit, now);
            unit = now;
            __syncwarp();
            if (j && __any_sync(~0u, by != 1.0f)) {
#pragma unroll 1
                for (uint32_t i = 0; i < columns; i += 32) {
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
            // Exponents are relative to the unit where that is near the largest p's, so that a weight is p times a scale; else to the largest p, and a
            // weight is multiplied once more. (Near: no sum of p passes fp32, and p of 2^-100 of the largest are numbers.)
            const bool near = __all_sync(~0u, (from - unit >= -26.0f && from - unit <= 60.0f) || ref == -INFINITY);
            const float base = near && ref != -INFINITY ? unit : from;
            const float2 minus = make_float2(-base, -base);
            float2 sum = make_float2(0.0f, 0.0f), more = sum;
            auto weigh = [&](auto once_more, float each_is) {
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    float x[32];
                    read(x, i);
                    uint32_t w[16];
#pragma unroll
                    for (uint32_t k = 0; k < 32; k += 4) {
                        const float by_f = factor(32u * i + k / 16u * 16u);
                        const float4 c = Group == 1 ? reinterpret_cast<const float4*>(value)[8u * i + k / 4] : make_float4(value[32u * i + k / 16u * 16u], 0.0f, 0.0f, 0.0f);
                        const float2 c0 = Group == 1 ? make_float2(c.x, c.y) : make_float2(c.x, c.x), c1 = Group == 1 ? make_float2(c.z, c.w) : c0;
                        const float2 f2 = make_float2(by_f, by_f);
                        const float2 d = fma2(make_float2(x[k], x[k + 1]), f2, minus), e = fma2(make_float2(x[k + 2], x[k + 3]), f2, minus);
                        const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y)), q = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                        sum = add2(sum, p);
                        more = add2(more, q);
                        float2 y = mul2(p, c0), z = mul2(q, c1);
                        if constexpr (decltype(once_more)::value) {
                            y = mul2(y, make_float2(each_is, each_is));
                            z = mul2(z, make_float2(each_is, each_is));
                        }
                        w[k / 2] = pair_of(y.x, y.y);
                        w[k / 2 + 1] = pair_of(z.x, z.y);
                    }
                    tmem_write16(scores + 16u * i, w); // (over scores of this thread's that have been read twice)
                }
            };
            if (near)
                weigh(std::false_type{}, 1.0f);
            else
                weigh(std::true_type{}, ex2_approx(from - unit)); // (0 where there is no weight yet)
            l += ((sum.x + sum.y) + (more.x + more.y)) * ex2_approx(base - from);
            __syncwarp();
            tmem_written();
            tc_fence_before();
            mbar_arrive(&s.p_full[t]);
            __syncwarp();
        }
        alive = alive && await(s, &s.o_full[t], outputs & 1u);
        ++outputs;
        __syncwarp();
        tc_fence_after();
        s.sum[half][row] = l;
        __syncwarp();
        named_barrier(pair, 64);
        l = half ? s.sum[0][row] + l : l + s.sum[1][row]; // (in the same order in both)
        for (uint32_t i = 0; i < s.n_mixed[which]; ++i) { // values that are NaN, of blocks that not all rows see
            const uint32_t* b = s.mixed[which][i];
            if (!(b[1] | b[2] | b[3] | b[4]))
                continue;
            for (uint32_t k = 0; k < kBlock; ++k) {
                const int32_t at_key = (int32_t)(b[0] * kBlock + k);
                if (((b[1 + k / 32u] >> (k & 31u)) & 1u) && at_key >= lo && at_key < hi)
                    l = __int_as_float(0x7fc00000);
            }
        }
        __syncwarp();
        const float worth = kv_worth(unit, ref);
        T* to = static_cast<T*>(a.out) + (g.seq.first + token) * a.out_ld + (uint64_t)head * D + half * columns;
        const float by = part ? worth : l == 0.0f ? 0.0f : worth / l;
#pragma unroll 1
        for (uint32_t i = 0; i < columns; i += 32) {
            float y[32];
            tmem_read32(y, out + i);
            if (real && part) {
#pragma unroll
                for (uint32_t k = 0; k < 32; ++k)
                    part[(half * columns + i + k) * kUnitRows + row] = y[k] * by; // (by column: lanes are rows)
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
        if (real && part && half == 0) {
            part[kUnitRows * D + row] = ref;
            part[kUnitRows * (D + 1u) + row] = l;
        }
        __syncwarp();
    }
};

template <typename T, uint32_t D, uint32_t Group>
__global__ void __launch_bounds__(kThreads, 1) kv_prompt_kernel(const KvAttendArgs a)
{
    extern __shared__ unsigned char raw[];
    __shared__ Shared s;
    Ring<D> ring;
    ring.base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    const uint32_t tid = threadIdx.x, warp = tid / 32u;
    if (tid == 0) {
        mbar_init(&s.q_full, 2u * kUnitRows);
        mbar_init(&s.q_empty, 1);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&s.k_full[i], 1);
            mbar_init(&s.k_empty[i], 1);
            mbar_init(&s.v_full[i], 1);
            mbar_init(&s.v_empty[i], 1);
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], 2u * kTileRows);
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
            g.see_to = top < 0 ? 0u : min((uint32_t)top, g.seq.keys);
            g.see_from = a.window && last > (int32_t)a.window ? (uint32_t)last - a.window : 0u;
            role(g, g.whole() ? nullptr : a.parts + (uint64_t)g.place(blockIdx.x) * (kUnitRows * (D + 2u)));
        }
    };
    if (blockIdx.x < found.ctas) {
        if (tid < kConvert) {
            Softmax<T, D, Group> x;
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

template <typename T, uint32_t D, uint32_t Group>
cudaError_t launch(const KvAttendArgs& a, cudaStream_t stream)
{
    constexpr uint32_t smem = Ring<D>::bytes + 1024u;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = set_once(done, kv_prompt_kernel<T, D, Group>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess)
        return e;
    kv_prompt_kernel<T, D, Group><<<kPromptCtas, kThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, uint32_t D>
cudaError_t launch_group(const KvAttendArgs& a, cudaStream_t stream)
{
    return a.c.page_size % 16u ? launch<T, D, 1>(a, stream) : launch<T, D, 16>(a, stream);
}

} // namespace

cudaError_t launch_kv_prompt(const KvAttendArgs& a, int type, cudaStream_t stream)
{
    if (type == MK_BF16)
        return a.c.dim == 128u ? launch_group<__nv_bfloat16, 128>(a, stream) : launch_group<__nv_bfloat16, 64>(a, stream);
    return a.c.dim == 128u ? launch_group<__half, 128>(a, stream) : launch_group<__half, 64>(a, stream);
}

} // namespace mk
