// The head with the requests' low-rank adapters beside it (mk_head_logits in include/mako_b200.h):
//     logits[t][v] = weight[v] . hidden[t] + up[a][v] . inner[t],   inner[t] = scale[a] (down[a] hidden[t]),   a = adapter[t]
// Two launches. The first brings the rows into the order of their adapters (a copy of the hidden states, a few MB at most) and
// forms `inner`, a CTA per row. The second streams the weight matrix once past the rows: it is what bounds a decode step (1.06 GB
// at 129280 x 4096), so every CTA has an equal share of the vocabulary, a run of columns of the logits in steps of 16, and keeps
// as much of it on the way as shared memory holds. Measured at 129280 x 4096, bf16, replayed from a graph: 165 us for a row with an
// adapter of rank 16 (0.99 of the rate of a copy), 199 for 64 rows with 16 of them; without adapters 168 for 64 rows, 200 for 128, 219 for
// 160, 253 for 192, 304 for 256, where what an SM takes in from L2 (about 65 GB/s) bounds it, 708 for 512; 429 for 320 rows of 151552, with
// 8 adapters of rank 64 692. (The first launch is 7 to 31 us of these, and hides nowhere: a CTA of the second has nearly all of an SM's
// registers, so that it starts where none of the first is left.)
//
// A tile is 128 vocabulary rows (the MMA's M, a lane of tensor memory each) by the batch's rows (its N, padded to 16). Batches of
// few rows take two or four vocabulary tiles side by side, so that the hidden states' tile, which comes from L2 every time, is
// read once for all of them. Three warps copy tiles in, one issues the MMAs, eight drain tensor memory.
//
// Precision: the tensor core's fp32 accumulator truncates. Of a step of 16 products each loses what lies below a quarter of an ulp of the
// largest among them and the accumulator, their sum what lies below an ulp; where all are of one sign that adds up to 7.9e-6 of a sum of
// 4096 terms in bf16, 2.3e-5 in fp16, whose products have more bits. So a run of 512 terms goes into one of two accumulators (2.3e-7 and
// 2.4e-6 then; of terms of either sign 4.7e-7 and 6.4e-7 of a logit, through one accumulator 4.4e-6) and is added in registers, rounding to
// nearest, while the next run goes into the other. `inner` stays in fp32; its products with `up` are FMAs of the draining warps,
// 16 or 32 ranks at a time between the runs: rows of one adapter stand side by side, so that a lane's piece of `up` is loaded once for
// all of them. (As MMAs they would want `inner` cut to 16 bits, and one adapter's infinite weight would reach other rows as 0 x inf.)
#include "round_ops.h"
#include "tcgen05.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mk {
namespace {

constexpr uint32_t kBlockK = 64;                   // elements of the contraction in a tile: 128 bytes
constexpr uint32_t kRunBlocks = 8;                 // tiles that go into one accumulator
constexpr uint32_t kTileV = 128, kGroupV = 16;     // vocabulary rows of a tile; of a CTA's share, a multiple
constexpr uint32_t kTileBytes = kTileV * kBlockK * 2;
constexpr uint32_t kWeightWarps = 2;                // that copy weights; before them one issues products, one copies rows
constexpr uint32_t kDrainWarps = 8, kFirstDrain = 4, kHeadThreads = 32 * (kFirstDrain + kDrainWarps);
constexpr int kRankStep = 16, kWideStep = 32;      // ranks that a lane holds of `up` at a time; where few rows leave registers for more
constexpr uint32_t kWideRows = 96;
constexpr uint32_t kDeltas = 16;                   // columns that the adapters' part is formed for at a time
constexpr uint32_t kMaxColumns = 256;              // of one of two accumulators: vocabulary tiles x rows
constexpr uint32_t kPairRows = 160;                // of two tiles side by side: one accumulator, what the draining warps have registers for
constexpr uint32_t kMaxStages = 16;
constexpr uint32_t kRingBytes = 178 * 1024;

__device__ __forceinline__ float2 pair_to_float(__nv_bfloat162 x) { return __bfloat1622float2(x); }
__device__ __forceinline__ float2 pair_to_float(__half2 x) { return __half22float2(x); }
template <typename T>
struct Type;
template <>
struct Type<__nv_bfloat16> {
    using pair = __nv_bfloat162;
    static constexpr bool bf16 = true;
};
template <>
struct Type<__half> {
    using pair = __half2;
    static constexpr bool bf16 = false;
};

// Eight elements as four pairs of floats.
template <typename T>
__device__ __forceinline__ void load8(float2 (&x)[4], const T* p)
{
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = pair_to_float(*reinterpret_cast<const typename Type<T>::pair*>(&w[i]));
}

// Where the rows go when they stand in the order of their adapters (rows without one last), and what the adapters' down
// projections leave of them. All indexed by the new place.
struct HeadOrder {
    void* hidden;   // [rows][dim]
    int32_t* row;   // which row stands here
    int32_t* adapter; // its adapter, or -1
    float* inner;   // [rows][kHeadMaxRank]; zeros where there is no adapter
};

// A CTA per row: its place is the number of rows that come before it; two dot products at a time per warp.
template <typename T>
__global__ void __launch_bounds__(256) head_inner_kernel(const mk_head h, const T* hidden, uint64_t hidden_ld,
                                                         const int32_t* adapter, uint32_t rows, const HeadOrder o)
{
    griddep_launch_dependents();
    __shared__ uint32_t s_before[8];
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, w = tid / 32u;
    auto key = [&](uint32_t i) {
        const uint32_t a = (uint32_t)adapter[i];
        return a < h.n_adapters ? a : ~0u;
    };
    const uint32_t a = key(row);
    uint32_t before = 0;
    for (uint32_t i = tid; i < rows; i += 256u) {
        const uint32_t b = key(i);
        before += b < a || (b == a && i < row);
    }
    before = __reduce_add_sync(~0u, before);
    if (lane == 0)
        s_before[w] = before;
    __syncthreads();
    uint32_t place = 0;
    for (int i = 0; i < 8; ++i)
        place += s_before[i];
    const T* x = hidden + row * hidden_ld;
    T* to = static_cast<T*>(o.hidden) + (size_t)place * h.dim;
    for (uint32_t i = tid * 8u; i < h.dim; i += 256u * 8u)
        *reinterpret_cast<uint4*>(to + i) = __ldg(reinterpret_cast<const uint4*>(x + i));
    if (tid == 0) {
        o.row[place] = (int32_t)row;
        o.adapter[place] = (int32_t)a;
    }
    float* out = o.inner + (size_t)place * kHeadMaxRank;
    if (a == ~0u) {
        if (tid < kHeadMaxRank)
            out[tid] = 0.0f;
        return;
    }
    const float scale = h.scale ? h.scale[a] : 1.0f;
    for (uint32_t r = 2u * w; r < h.rank; r += 16u) { // (the rank is even)
        const T* d = static_cast<const T*>(h.down) + ((size_t)a * h.rank + r) * h.dim;
        float2 sum[2][4] = {};
#pragma unroll 4
        for (uint32_t i = lane * 8u; i < h.dim; i += 256u) {
            float2 p[4], q0[4], q1[4];
            load8(p, x + i);
            load8(q0, d + i);
            load8(q1, d + h.dim + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                sum[0][k] = fma2(p[k], q0[k], sum[0][k]);
                sum[1][k] = fma2(p[k], q1[k], sum[1][k]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                y += sum[j][k].x + sum[j][k].y;
#pragma unroll
            for (uint32_t k = 16; k; k >>= 1)
                y += __shfl_xor_sync(~0u, y, k);
            if (lane == 0)
                out[r + j] = scale * y;
        }
    }
}

struct HeadArgs {
    mk_head h;
    HeadOrder order; // of no meaning without adapters
    float* logits;
    uint64_t ld;
    uint32_t rows;
    uint32_t n;            // rows of a tile, a multiple of 16
    uint32_t side;         // vocabulary tiles side by side: 4, 2 or 1
    uint32_t bufs;         // accumulators of side * n columns: two of up to 256, or one of up to 320
    uint32_t spread;       // row tiles that CTAs side by side have at the same time
    uint32_t turn;         // steps of the contraction that a vocabulary tile is copied for before the next one's turn: 1, 2 or 4
    uint32_t w_slots, x_slots;
};

struct HeadShared {
    uint64_t w_full[kMaxStages], w_empty[kMaxStages], x_full[kMaxStages], x_empty[kMaxStages];
    uint64_t acc_full[2], acc_empty[2];
    uint32_t tmem;
    int failed;
    int32_t row[kMaxColumns], adapter[kMaxColumns]; // of the tile's columns
};

// And what the adapters' part needs, where a draining thread has so many vocabulary tiles.
template <int Tiles, int Step>
struct DrainShared {
    float4 inner[Step == kWideStep ? kWideRows : Tiles == 2 ? kPairRows : kMaxColumns][Step / 4];
    float delta[kDrainWarps][kDeltas][32][Tiles]; // each thread's own; kept here because registers take no running index
};

// A ring's place: slot and the parity its barriers complete with next.
struct Place {
    uint32_t slot = 0, parity = 0;
    __device__ void next(uint32_t n)
    {
        if (++slot == n) {
            slot = 0;
            parity ^= 1u;
        }
    }
};

// Waits, but not for ever: one that lasts two seconds, in any warp, ends all. (Probes without a suspend-time hint: with one of
// 20 us a step of the contraction took 0.65 us whatever its size.)
__device__ __forceinline__ bool await(HeadShared& s, uint64_t* bar, uint32_t parity)
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

// A CTA's rings and its share of the vocabulary: [v_from, v_end) is copied, [v_from, v_to) is written.
struct Share {
    unsigned char *ring, *x_ring;
    uint32_t x_bytes, k_blocks, v_from, v_end, v_to;
    uint32_t t_from, t_step; // its row tiles
};

// A draining thread has a lane, which is a vocabulary row, of one or two tiles side by side, and up to Rows of the batch's rows in each.
// Two where they fit, because what the adapters' part costs is reading `inner`: a float4 that all lanes of a warp share takes shared
// memory, of which the products' operands want all but a tenth, as long as 32 of them, and so serves two vocabulary rows (320 rows with
// adapters of rank 64 at 151552 x 4096: 690 us, with one tile a thread 868; without adapters 435).
template <typename T, int Tiles, int Rows, int Step>
__device__ __forceinline__ void drain(const HeadArgs& a, HeadShared& s, DrainShared<Tiles, Step>& own, const Share& c)
{
    const uint32_t v_from = c.v_from, v_to = c.v_to;
    const uint32_t tid = threadIdx.x - 32u * kFirstDrain, w = tid / 32u, lane = tid & 31u;
    const uint32_t quarter = w & 3u; // of the lanes, the one that this warp may read
    // four tiles: two for each four warps; fewer: half of the rows for each
    const uint32_t g0 = a.side == 4u ? w / 4u * 2u : 0u, m = a.side == 4u ? a.n : a.n / 2u, row0 = a.side == 4u ? 0u : w / 4u * m;
    const uint32_t k_blocks = (a.h.dim + kBlockK - 1) / kBlockK, runs = (k_blocks + kRunBlocks - 1) / kRunBlocks;
    const uint32_t steps = a.h.n_adapters ? (a.h.rank + Step - 1) / Step : 0u;
    constexpr uint32_t blocks = Rows / kDeltas;
    const uint32_t units = steps * blocks;
    const uint32_t tmem = s.tmem + ((quarter * 32u) << 16) + g0 * a.n + row0;
    const T* up = static_cast<const T*>(a.h.up);
    float acc[Tiles][Rows];
    uint32_t buf = 0, parity = 0;
    bool alive = true;
    griddep_wait(); // for the rows' order and `inner`
    for (uint32_t t0 = c.t_from; t0 < a.rows; t0 += c.t_step) {
        named_barrier(1, kDrainWarps * 32);
        if (tid < a.n) {
            const bool real = t0 + tid < a.rows;
            s.row[tid] = !real ? -1 : steps ? a.order.row[t0 + tid] : (int32_t)(t0 + tid);
            s.adapter[tid] = real && steps ? a.order.adapter[t0 + tid] : -1;
        }
        named_barrier(1, kDrainWarps * 32);
        uint32_t turns[(Rows + 31) / 32]; // rows whose adapter is another than the one's before
#pragma unroll
        for (int k = 0; k < (Rows + 31) / 32; ++k) {
            const uint32_t i = 32u * k + lane, t = row0 + i;
            turns[k] = __ballot_sync(~0u, i < m && (i == 0 || s.adapter[t] != s.adapter[t - 1u]));
        }
        for (uint32_t v0 = v_from; v0 < v_to; v0 += a.side * kTileV) {
            const uint32_t v = v0 + g0 * kTileV + quarter * 32u + lane; // in the first of its tiles
#pragma unroll
            for (int i = 0; i < Rows; ++i)
                acc[0][i] = acc[Tiles - 1][i] = 0.0f;
            uint32_t unit = 0;
            for (uint32_t run = 0; run < runs; ++run) {
                alive = alive && await(s, &s.acc_full[buf], parity); // a warp that gave up still meets the others' barriers
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < Rows; i += 32 / Tiles) { // (columns behind the rows that are its own hold anything, and are not written)
                    const int j = Tiles == 2 ? i : i + 16;
                    float x[2][16];
                    tmem_load16(x[0], tmem + buf * kMaxColumns + i);
                    tmem_load16(x[1], tmem + buf * kMaxColumns + (Tiles == 2 ? a.n : 0u) + j);
                    tmem_wait(x[0], x[1]);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        acc[0][i + k] += x[0][k];
                        acc[Tiles - 1][j + k] += x[1][k];
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&s.acc_empty[buf]);
                buf = buf + 1u == a.bufs ? 0u : buf + 1u;
                parity ^= buf == 0;
                // this run's part of the adapters' work, which is Step ranks of 16 rows at a time
                for (const uint32_t until = ((run + 1u) * units + runs - 1u) / runs; unit < until;) {
                    const uint32_t r = unit / blocks * Step, left = a.h.rank - r, from = unit % blocks;
                    const uint32_t to = min(blocks, from + until - unit);
                    unit += to - from;
                    if (from == 0 && (steps > 1 || v0 == v_from)) {
                        named_barrier(1, kDrainWarps * 32); // the ranks before these have been used
                        for (uint32_t i = tid; i < a.n * (Step / 4); i += kDrainWarps * 32) {
                            const uint32_t t = i / (Step / 4), q = i % (Step / 4);
                            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (t0 + t < a.rows && q * 4u < left)
                                y = __ldg(reinterpret_cast<const float4*>(a.order.inner + (size_t)(t0 + t) * kHeadMaxRank + r) + q);
                            own.inner[t][q] = y;
                        }
                        named_barrier(1, kDrainWarps * 32);
                    }
#pragma unroll
                    for (int block = 0; block < (int)blocks; ++block) {
                        if ((uint32_t)block < from || (uint32_t)block >= to || (uint32_t)block * kDeltas >= m)
                            continue;
                        uint32_t t = row0 + block * kDeltas, c = 0;
                        if (s.adapter[t] < 0) // nor has a row behind it an adapter
                            continue;
                        const uint32_t turn = (turns[block / 2] >> (block % 2 * 16)) | 1u, last = min(kDeltas, m - block * kDeltas);
                        while (c < last) {
                            const int32_t ad = s.adapter[t];
                            float2 x[Tiles][Step / 2];
#pragma unroll
                            for (int g = 0; g < Tiles; ++g) {
#pragma unroll
                                for (int i = 0; i < (int)Step / 2; ++i)
                                    x[g][i] = make_float2(0.0f, 0.0f);
                                if (ad >= 0 && v + g * kTileV < v_to) {
                                    const T* p = up + ((size_t)ad * a.h.n_vocab + v + g * kTileV) * a.h.rank + r;
                                    load8(*reinterpret_cast<float2(*)[4]>(&x[g][0]), p);
#pragma unroll
                                    for (int i = 8; i < Step; i += 8)
                                        if (left > (uint32_t)i)
                                            load8(*reinterpret_cast<float2(*)[4]>(&x[g][i / 2]), p + i);
                                }
                            }
                            const uint32_t later = (turn >> c) >> 1;
                            const uint32_t end = later ? min(c + (uint32_t)__ffs(later), last) : last;
                            const float4(*y)[Step / 4] = &own.inner[t];
                            t += end - c;
#pragma unroll 2
                            for (; c < end; ++c, ++y) {
                                float2 d[Tiles] = {}, e[Tiles] = {};
#pragma unroll
                                for (int i = 0; i < (int)Step / 4; ++i) {
                                    const float4 z = (*y)[i];
#pragma unroll
                                    for (int g = 0; g < Tiles; ++g) {
                                        d[g] = fma2(x[g][2 * i], make_float2(z.x, z.y), d[g]);
                                        e[g] = fma2(x[g][2 * i + 1], make_float2(z.z, z.w), e[g]);
                                    }
                                }
#pragma unroll
                                for (int g = 0; g < Tiles; ++g)
                                    own.delta[w][c][lane][g] = (d[g].x + e[g].x) + (d[g].y + e[g].y);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < (int)kDeltas; ++k) { // (behind the last row what an earlier block left)
#pragma unroll
                            for (int g = 0; g < Tiles; ++g)
                                acc[g][block * (int)kDeltas + k] += own.delta[w][k][lane][g];
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < Rows; ++k) {
                const int32_t row = (uint32_t)k < m ? s.row[row0 + k] : -1;
                if (row >= 0) {
                    float* p = a.logits + (size_t)row * a.ld + v;
#pragma unroll
                    for (int g = 0; g < Tiles; ++g)
                        if (v + g * kTileV < v_to)
                            p[g * kTileV] = acc[g][k];
                }
            }
        }
    }
}

// One of kWeightWarps threads that copy weights: a tile each in turn. (A thread takes about 150 cycles from one copy to the next.)
__device__ __forceinline__ void copy_weights(const HeadArgs& a, HeadShared& s, const Share& c, const CUtensorMap* w_map,
                                             const CUtensorMap* w_small, uint32_t mine)
{
    const uint64_t policy = a.spread > 1 ? l2_evict_last() : l2_evict_first(); // do other CTAs read them too?
    Place w;
    uint32_t turn = 0;
    for (uint32_t t0 = c.t_from; t0 < a.rows; t0 += c.t_step)
        for (uint32_t v0 = c.v_from; v0 < c.v_end; v0 += a.side * kTileV)
            for (uint32_t k0 = 0; k0 < c.k_blocks; k0 += a.turn)
                for (uint32_t v = v0; v < c.v_end && v < v0 + a.side * kTileV; v += kTileV)
                    for (uint32_t k = k0; k < c.k_blocks && k < k0 + a.turn; ++k) {
                        if (turn == mine) {
                            if (!await(s, &s.w_empty[w.slot], w.parity ^ 1u))
                                return;
                            unsigned char* to = c.ring + w.slot * kTileBytes;
                            const uint32_t left = c.v_end - v;
                            if (left >= kTileV) {
                                mbar_arrive_expect_tx(&s.w_full[w.slot], kTileBytes);
                                tma_load_2d(to, w_map, (int32_t)(k * kBlockK), (int32_t)v, &s.w_full[w.slot], policy);
                            } else { // the share's end, in steps of 16 rows; what lies behind them in the slot has no part
                                mbar_arrive_expect_tx(&s.w_full[w.slot], left * kBlockK * 2);
                                for (uint32_t i = 0; i < left; i += kGroupV)
                                    tma_load_2d(to + i * kBlockK * 2, w_small, (int32_t)(k * kBlockK), (int32_t)(v + i), &s.w_full[w.slot],
                                                policy);
                            }
                        }
                        w.next(a.w_slots);
                        turn = turn + 1u == kWeightWarps ? 0u : turn + 1u;
                    }
}

// And the one that copies hidden states, once their order is there.
__device__ __forceinline__ void copy_rows(const HeadArgs& a, HeadShared& s, const Share& c, const CUtensorMap* x_map)
{
    const uint64_t policy = l2_evict_last();
    Place x;
    griddep_wait();
    for (uint32_t t0 = c.t_from; t0 < a.rows; t0 += c.t_step)
        for (uint32_t v0 = c.v_from; v0 < c.v_end; v0 += a.side * kTileV)
            for (uint32_t k0 = 0; k0 < c.k_blocks; k0 += a.turn) {
                if (!await(s, &s.x_empty[x.slot], x.parity ^ 1u))
                    return;
                const uint32_t steps = min(a.turn, c.k_blocks - k0);
                unsigned char* to = c.x_ring + x.slot * a.turn * c.x_bytes;
                mbar_arrive_expect_tx(&s.x_full[x.slot], steps * c.x_bytes);
                for (uint32_t i = 0; i < steps; ++i)
                    tma_load_2d(to + i * c.x_bytes, x_map, (int32_t)((k0 + i) * kBlockK), (int32_t)t0, &s.x_full[x.slot], policy);
                x.next(a.x_slots);
            }
}

// The one that issues products.
template <typename T>
__device__ __forceinline__ void issue(const HeadArgs& a, HeadShared& s, const Share& c)
{
    const uint32_t desc = mma_f16_desc(Type<T>::bf16, a.n), tmem = s.tmem;
    const uint64_t w_desc = smem_tile_desc(c.ring), x_desc = smem_tile_desc(c.x_ring);
    Place w, x;
    uint32_t buf = 0, parity = 0;
    for (uint32_t t0 = c.t_from; t0 < a.rows; t0 += c.t_step)
        for (uint32_t v0 = c.v_from; v0 < c.v_end; v0 += a.side * kTileV) {
            const uint32_t tiles = min(a.side, (c.v_end - v0 + kTileV - 1u) / kTileV);
            for (uint32_t k0 = 0; k0 < c.k_blocks; k0 += a.turn) {
                const uint32_t steps = min(a.turn, c.k_blocks - k0);
                uint32_t add = k0 % kRunBlocks != 0;
                if (!add && !await(s, &s.acc_empty[buf], parity ^ 1u))
                    return;
                if (!await(s, &s.x_full[x.slot], x.parity))
                    return;
                const uint64_t b0 = x_desc + (x.slot * a.turn * c.x_bytes >> 4);
                uint32_t d = tmem + buf * kMaxColumns;
                for (uint32_t g = 0; g < tiles; ++g, d += a.n) {
                    uint64_t b = b0;
                    uint32_t more = add;
                    for (uint32_t i = 0; i < steps; ++i, b += c.x_bytes >> 4) {
                        if (!await(s, &s.w_full[w.slot], w.parity))
                            return;
                        tc_fence_after();
                        const uint64_t t = w_desc + (w.slot * kTileBytes >> 4);
                        mma_f16(d, t, b, desc, more);
                        mma_f16(d, t + 2, b + 2, desc, true);
                        mma_f16(d, t + 4, b + 4, desc, true);
                        mma_f16(d, t + 6, b + 6, desc, true);
                        mma_commit(&s.w_empty[w.slot]);
                        w.next(a.w_slots);
                        more = 1;
                    }
                }
                mma_commit(&s.x_empty[x.slot]);
                x.next(a.x_slots);
                if ((k0 + steps) % kRunBlocks == 0 || k0 + steps == c.k_blocks) {
                    mma_commit(&s.acc_full[buf]);
                    buf = buf + 1u == a.bufs ? 0u : buf + 1u;
                    parity ^= buf == 0;
                }
            }
        }
}

template <typename T, int Tiles, int Rows, int Step>
__global__ void __launch_bounds__(kHeadThreads, 1)
    head_kernel(const HeadArgs a, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap w_small,
                const __grid_constant__ CUtensorMap x_map)
{
    extern __shared__ unsigned char raw[];
    __shared__ HeadShared s;
    __shared__ DrainShared<Tiles, Step> own;
    const uint32_t warp = threadIdx.x / 32u, groups = (a.h.n_vocab + kGroupV - 1) / kGroupV;
    Share c;
    c.ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    c.x_ring = c.ring + a.w_slots * kTileBytes;
    c.x_bytes = a.n * kBlockK * 2;
    c.k_blocks = (a.h.dim + kBlockK - 1) / kBlockK;
    const uint32_t shares = gridDim.x / a.spread, mine = blockIdx.x / a.spread;
    c.v_from = (uint32_t)((uint64_t)groups * mine / shares) * kGroupV;
    c.v_end = (uint32_t)((uint64_t)groups * (mine + 1u) / shares) * kGroupV;
    c.t_from = blockIdx.x % a.spread * a.n;
    c.t_step = a.spread * a.n;
    c.v_to = min(c.v_end, a.h.n_vocab);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kMaxStages; ++i) {
            mbar_init(&s.w_full[i], 1);
            mbar_init(&s.w_empty[i], 1);
            mbar_init(&s.x_full[i], 1);
            mbar_init(&s.x_empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&s.acc_full[i], 1);
            mbar_init(&s.acc_empty[i], kDrainWarps);
        }
        s.failed = 0;
        fence_barrier_init();
    }
    if (warp == 1)
        tmem_alloc_all(&s.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // 168 registers a thread at launch: 128 threads give up what 256 that drain take (128 x 40 + 256 x 232 = 384 x 168)
    if (warp >= kFirstDrain) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        drain<T, Tiles, Rows, Step>(a, s, own, c);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (threadIdx.x == 0)
            issue<T>(a, s, c);
        else if (threadIdx.x == 32)
            copy_rows(a, s, c, &x_map);
        else if (threadIdx.x == 64 || threadIdx.x == 96)
            copy_weights(a, s, c, &w_map, &w_small, threadIdx.x / 32u - 2u);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (s.failed) { // never seen: copies and products in flight end within this, and the share's logits say what happened
        for (int i = 0; i < 2000; ++i)
            __nanosleep(1000);
        for (uint32_t t = 0; t < a.rows; ++t) // (of all rows: which ones were this CTA's is in what may have failed)
            for (uint32_t v = c.v_from + threadIdx.x; v < c.v_to; v += kHeadThreads)
                a.logits[(size_t)t * a.ld + v] = __int_as_float(0x7fc00000);
        __syncthreads();
    }
    if (warp == 1)
        tmem_free_all(s.tmem);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encoder(EncodeTiled& f)
{
    static std::atomic<void*> found{nullptr};
    void* p = found.load(std::memory_order_relaxed);
    if (!p) {
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess)
            return e;
        if (!p || q != cudaDriverEntryPointSuccess)
            return cudaErrorNotSupported;
        found.store(p, std::memory_order_relaxed);
    }
    f = reinterpret_cast<EncodeTiled>(p);
    return cudaSuccess;
}

// A row-major matrix of 16-bit elements in boxes of 64 elements by `box` rows.
bool encode(EncodeTiled f, CUtensorMap* map, bool bf16, const void* base, uint64_t cols, uint64_t rows, uint64_t ld, uint32_t box)
{
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
    const cuuint32_t boxes[2] = {kBlockK, box}, steps[2] = {1, 1};
    return f(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides,
             boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int Tiles, int Rows, int Step>
cudaError_t launch_tiles(const HeadArgs& a, uint32_t grid, bool behind_inner, const CUtensorMap* maps, cudaStream_t stream)
{
    const size_t smem = kRingBytes + 1024;
    static const bool split_fits = [] { // the registers that the warps share out among themselves are those of the launch
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, head_kernel<T, Tiles, Rows, Step>) == cudaSuccess && f.numRegs == 168;
    }();
    if (!split_fits)
        return cudaErrorInvalidKernelImage;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = set_once(done, head_kernel<T, Tiles, Rows, Step>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(kHeadThreads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = behind_inner ? 1 : 0;
    return cudaLaunchKernelEx(&c, head_kernel<T, Tiles, Rows, Step>, a, maps[0], maps[1], maps[2]);
}

template <typename T>
cudaError_t launch(const mk_head& h, const void* hidden, uint64_t hidden_ld, const int32_t* adapter, uint32_t rows,
                   const HeadScratch& scratch, float* logits, uint64_t ld, cudaStream_t stream)
{
    EncodeTiled f;
    cudaError_t e = encoder(f);
    if (e != cudaSuccess)
        return e;
    HeadArgs a;
    a.h = h;
    a.order.hidden = scratch.hidden;
    a.order.row = scratch.ints;
    a.order.adapter = scratch.ints + rows;
    a.order.inner = scratch.inner;
    a.logits = logits;
    a.ld = ld;
    a.rows = rows;
    // What the ring carries for a step of 64 of the contraction and 128 vocabulary rows is 16 KB of weights and, over the tiles side
    // by side, the rows' 128 bytes each; rows by the 160 in CTAs side by side, which read the same weights at the same time, carry the
    // least beyond 256. (From 161 to 256 one tile of all rows is better: 192 rows 253 us, as two of 96 353; 256 rows 304, as two of 128 362.)
    const uint32_t tiles = rows <= kMaxColumns ? 1u : (rows + kPairRows - 1) / kPairRows;
    a.n = ((rows + tiles - 1) / tiles + 15u) & ~15u;
    a.side = a.n <= kMaxColumns / 4 ? 4u : a.n <= kPairRows ? 2u : 1u;
    a.bufs = a.side * a.n <= kMaxColumns ? 2u : 1u;
    a.spread = tiles < 8u ? tiles : 8u;
    const uint32_t x_bytes = a.n * kBlockK * 2;
    // What a step costs beside its bytes is the issuing thread's time, barriers mostly: steps in turns of four share one for the rows, and
    // the weights come in pieces of 512 bytes a row. In turns of 1, 2, 4 a call without adapters of 129280 x 4096 took 187, 163, 158 us
    // for one row, 194, 169, 167 for 64, 232, 199, 230 for 128 (whose rows fill the ring), 316, 305, 304 for 256.
    a.turn = a.n <= kMaxColumns / 4 ? 4u : 2u;
    // As deep a ring of tiles as fits: of rows two turns at least, of weights a tile for each of their warps (with fewer a warp could
    // be two rounds of the ring ahead, and take a barrier's phase for another).
    a.x_slots = a.w_slots = 0;
    for (uint32_t best = 0; a.turn && !best; a.turn /= best ? 1u : 2u)
        for (uint32_t x = 2; x <= kMaxStages && x * a.turn * x_bytes < kRingBytes; ++x) {
            uint32_t w = (kRingBytes - x * a.turn * x_bytes) / kTileBytes;
            w = w > kMaxStages ? kMaxStages : w;
            const uint32_t deep = w < x * a.turn * a.side ? w : x * a.turn * a.side;
            if (w >= kWeightWarps && deep > best) {
                best = deep;
                a.x_slots = x;
                a.w_slots = w;
            }
        }
    if (a.w_slots < kWeightWarps || a.x_slots * a.turn * x_bytes + a.w_slots * kTileBytes > kRingBytes)
        return cudaErrorInvalidConfiguration;
    CUtensorMap maps[3];
    constexpr bool bf16 = Type<T>::bf16;
    if (!encode(f, &maps[0], bf16, h.weight, h.dim, h.n_vocab, h.dim, kTileV) ||
        !encode(f, &maps[1], bf16, h.weight, h.dim, h.n_vocab, h.dim, kGroupV) ||
        !encode(f, &maps[2], bf16, h.n_adapters ? scratch.hidden : hidden, h.dim, rows, h.n_adapters ? h.dim : hidden_ld, a.n))
        return cudaErrorInvalidValue;
    if (h.n_adapters)
        head_inner_kernel<T><<<rows, 256, 0, stream>>>(h, static_cast<const T*>(hidden), hidden_ld, adapter, rows, a.order);
    e = cudaGetLastError();
    if (e != cudaSuccess)
        return e;
    const uint32_t groups = (h.n_vocab + kGroupV - 1) / kGroupV, most = 148u / a.spread;
    const uint32_t grid = (groups < most ? groups : most) * a.spread;
    const uint32_t half = a.side == 4u ? a.n : a.n / 2u;
    const bool behind = h.n_adapters != 0;
    // What rows of many adapters wait for is `up`, once for every adapter and step of ranks: 64 rows, 16 adapters of rank 64 at 129280 x 4096
    // by steps of 16 422 us, of 32 313; of rank 32 227 and 217; 96 rows with 4 of rank 128 394 and 336; 16 rows with 4 of rank 64 193 and
    // 194; a row with one 176 and 178. (16 rows with an adapter of rank 64 each are on the wrong side of the bound: 389 and 308.)
    if (h.n_adapters && h.rank > (uint32_t)kRankStep && a.n > 16u && a.n <= kWideRows)
        return half <= 32 ? launch_tiles<T, 2, 32, kWideStep>(a, grid, behind, maps, stream)
               : half <= 48 ? launch_tiles<T, 2, 48, kWideStep>(a, grid, behind, maps, stream)
                            : launch_tiles<T, 2, 64, kWideStep>(a, grid, behind, maps, stream);
    return half <= 16 ? launch_tiles<T, 2, 16, kRankStep>(a, grid, behind, maps, stream)
           : half <= 32 ? launch_tiles<T, 2, 32, kRankStep>(a, grid, behind, maps, stream)
           : half <= 48 ? launch_tiles<T, 2, 48, kRankStep>(a, grid, behind, maps, stream)
           : half <= 64 ? launch_tiles<T, 2, 64, kRankStep>(a, grid, behind, maps, stream)
           : half <= 80 ? launch_tiles<T, 2, 80, kRankStep>(a, grid, behind, maps, stream)
           : half <= 96 ? launch_tiles<T, 1, 96, kRankStep>(a, grid, behind, maps, stream)
                        : launch_tiles<T, 1, 128, kRankStep>(a, grid, behind, maps, stream);
}

} // namespace

cudaError_t launch_head_logits(const mk_head& h, const void* hidden, uint64_t hidden_ld, const int32_t* adapter, uint32_t rows,
                               const HeadScratch& scratch, float* logits, uint64_t ld, cudaStream_t stream)
{
    return h.type == MK_BF16 ? launch<__nv_bfloat16>(h, hidden, hidden_ld, adapter, rows, scratch, logits, ld, stream)
                             : launch<__half>(h, hidden, hidden_ld, adapter, rows, scratch, logits, ld, stream);
}

} // namespace mk
