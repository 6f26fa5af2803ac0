// Log-probabilities of given tokens, the entropy and the likeliest alternatives of whole distributions (mk_token_logprobs in
// include/mako_b200.h): every logit is read once.
//
// With c = log2(e) / temperature and any shift s a row's weights are w_i = 2^(c x_i - s); log2 of a probability is c x_t - s -
// log2(sum w), and the entropy in bits log2(sum w) - sum(w (c x - s)) / sum w. Each thread keeps (s, sum w, sum w (c x - s)) of its columns,
// s being c times the largest x so far, rounded: a shift that is a little off is as good as another as long as it is the same one
// everywhere, so that what the rounding of a large c x takes away does not reach the results.
//
// Alternatives: an x above `line` goes into a list of (x, id) in shared memory. The line is a lower bound of the k-th largest x that the
// CTA has seen: of the threads' largest ones in the first tile, then of the list's entries after 2, 4, 8, ... tiles, so that a row in
// no particular order has about k log2(tiles) entries. A row whose list runs over (an ascending one) is read again, in pieces of
// which each fits.
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
constexpr uint32_t kRankMax = kThreads;      // entries that are ranked against one another
constexpr uint32_t kMaxCluster = 8;
constexpr float kLeast = -200.0f;            // exponents are held above this: 2^-200 is nothing, and nothing times it is not NaN

using Key = unsigned long long;              // larger x first, then the lower id

__device__ __forceinline__ Key make_key(float x, uint32_t id) { return ((Key)order_key(x) << 32) | (uint32_t)~id; }
__device__ __forceinline__ float key_x(Key k) { return key_to_float((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_id(Key k) { return ~(uint32_t)k; }

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
    Sums<double> sums;     // (in 64 bits: c times a mask of the type's lowest value passes fp32)
    Sums<float> warp[kWarps];
    float largest[kThreads];
    uint32_t n;        // entries that were to go into the list
    uint32_t n_best;
    uint32_t allowed;  // not 0: the mask allows a token
    float line;
};

template <typename T>
struct Block { // 16 bytes of logits
    static constexpr uint32_t n = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void values(float (&x)[n]) const
    {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = y.x;
                x[2 * i + 1] = y.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};

// A CTA's columns of a row: blocks [from, to) of those that begin at the last 16-byte boundary in front of the row.
struct Columns {
    const uint4* base;
    uint32_t before;   // elements of the first block that are in front of the row
    uint32_t n_vocab;
    uint32_t from, to;
    const uint32_t* mask;
};

// Block b's logits, -inf where there is none, and where the mask allows none. The bits that say which there are go to `there`.
template <typename T, bool Mask>
__device__ __forceinline__ void columns_of(const Columns& c, uint32_t b, const Block<T>& block, float (&x)[Block<T>::n], uint32_t& there)
{
    constexpr uint32_t n = Block<T>::n;
    block.values(x);
    const int32_t first = (int32_t)(b * n) - (int32_t)c.before;
    there = (1u << n) - 1u;
    if (first < 0)
        there &= ~0u << -first;
    if (first + (int32_t)n > (int32_t)c.n_vocab)
        there &= first >= (int32_t)c.n_vocab ? 0u : (1u << (c.n_vocab - first)) - 1u;
    if (Mask && there) {
        const uint32_t at = first < 0 ? 0u : (uint32_t)first, word = at / 32u, last = (c.n_vocab - 1u) / 32u;
        const uint32_t bits = __funnelshift_r(__ldg(c.mask + word), word < last ? __ldg(c.mask + word + 1u) : 0u, at & 31u);
        there &= first < 0 ? bits << -first : bits;
    }
    if (Mask || there != (1u << n) - 1u) {
#pragma unroll
        for (uint32_t i = 0; i < n; ++i)
            x[i] = (there >> i) & 1u ? x[i] : -INFINITY;
    }
}

template <uint32_t N>
__device__ __forceinline__ float largest_of(const float (&x)[N])
{
    float m = x[0]; // (NaN loses)
#pragma unroll
    for (uint32_t i = 1; i < N; ++i)
        m = fmaxf(m, x[i]);
    return m;
}

template <uint32_t N>
__device__ __forceinline__ void add(Sums<float>& s, const float (&x)[N], float c, float most)
{
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
    for (uint32_t i = 0; i < N; i += 2) {
        float2 d = fma2(make_float2(x[i], x[i + 1]), c2, minus);
        d.x = fmaxf(d.x, kLeast); // NaN, -inf and what is masked too
        d.y = fmaxf(d.y, kLeast);
        const float2 w = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        w2.x += w.x;
        w2.y += w.y;
        d2 = fma2(w, d, d2);
    }
    s.w += w2.x + w2.y;
    s.wd += d2.x + d2.y;
}

// A lower bound of the k-th largest of n numbers (n >= k), by one warp: its upper 16 bits in the order of floats.
template <typename F>
__device__ float kth_bound(uint32_t n, uint32_t k, F value)
{
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t at = 0;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
        uint32_t count = 0;
        for (uint32_t i = lane; i < n; i += 32u)
            count += order_key(value(i)) >= (at | bit);
        if (__reduce_add_sync(~0u, count) >= k)
            at |= bit;
    }
    return at < order_key(-INFINITY) ? -INFINITY : key_to_float(at);
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

// The k largest of the list's first n keys in order, into `best`.
__device__ void rank_best(Shared& s, uint32_t n, uint32_t k)
{
    const uint32_t tid = threadIdx.x;
    if (n > kRankMax)
        n = keep_best(s, n, k);
    __syncthreads();
    const Key mine = tid < n ? s.list[tid] : 0;
    uint32_t rank = 0;
    if (tid < n)
        for (uint32_t i = 0; i < n; ++i)
            rank += s.list[i] > mine;
    if (tid < n && rank < k)
        s.best[rank] = mine;
    if (tid == 0)
        s.n_best = n < k ? n : k;
    __syncthreads();
}

// Puts block b's logits above the line into the list, as long as it has room.
template <uint32_t N>
__device__ __forceinline__ void put(Shared& s, const Columns& c, uint32_t b, const float (&x)[N], float line, bool also)
{
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
        if (x[i] > line || (also && x[i] == line && x[i] > -INFINITY)) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < kListCap)
                s.list[at] = make_key(x[i], b * N - c.before + i);
        }
}

template <typename T, bool Mask>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const mk_logprob_rows r, const LogprobOut o)
{
    constexpr uint32_t N = Block<T>::n;
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t slices = cluster.num_blocks(), slice = cluster.block_rank(), row = blockIdx.x / slices;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, k = r.n_top ? r.n_top : 1u;
    griddep_launch_dependents();
    if (tid == 0) {
        s.n = 0;
        s.allowed = 0;
    }
    griddep_wait();
    Columns c;
    const T* x0 = static_cast<const T*>(r.logits) + (size_t)row * r.ld;
    c.before = (uint32_t)((reinterpret_cast<uintptr_t>(x0) & 15u) / sizeof(T));
    c.base = reinterpret_cast<const uint4*>(x0 - c.before);
    c.n_vocab = r.n_vocab;
    c.mask = Mask ? r.mask + (size_t)row * r.mask_ld : nullptr;
    const uint32_t blocks = (c.before + r.n_vocab + N - 1) / N;
    c.from = (uint32_t)((uint64_t)blocks * slice / slices);
    c.to = (uint32_t)((uint64_t)blocks * (slice + 1u) / slices);
    const float t = r.temperature ? __ldg(r.temperature + row) : r.temperature_all;
    const bool greedy = !(t > 1e-30f && t < 1e30f);
    const float scale = greedy ? 1.0f : 1.44269504088896340736f / t;

    Sums<float> sums{-INFINITY, 0.0f, 0.0f};
    uint32_t any = 0, turn = 2;
    float line = -INFINITY;
    uint32_t tile = 0;
    for (uint32_t b0 = c.from; b0 < c.to; b0 += kThreads * kTileVecs, ++tile) {
        Block<T> block[kTileVecs];
#pragma unroll
        for (uint32_t j = 0; j < kTileVecs; ++j) {
            const uint32_t b = b0 + j * kThreads + tid;
            block[j].raw = b < c.to ? __ldcs(c.base + b) : make_uint4(0, 0, 0, 0);
        }
        if (tile == 0) { // what the line starts from
            float most = -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < kTileVecs; ++j) {
                const uint32_t b = b0 + j * kThreads + tid;
                if (b >= c.to)
                    continue;
                float x[N];
                uint32_t there;
                columns_of<T, Mask>(c, b, block[j], x, there);
                most = fmaxf(most, largest_of(x));
            }
            s.largest[tid] = most;
            __syncthreads();
            if (tid < 32u) {
                const float bound = kth_bound(kThreads, k, [&](uint32_t i) { return s.largest[i]; });
                if (lane == 0)
                    s.line = bound;
            }
            __syncthreads();
            line = s.line;
        } else if (tile == turn) {
            turn *= 2u;
            __syncthreads();
            if (tid < 32u) {
                const uint32_t n = min(s.n, kListCap);
                const float bound = n < k ? -INFINITY : kth_bound(n, k, [&](uint32_t i) { return key_x(s.list[i]); });
                if (lane == 0)
                    s.line = fmaxf(line, bound);
            }
            __syncthreads();
            line = s.line;
        }
#pragma unroll
        for (uint32_t j = 0; j < kTileVecs; ++j) {
            const uint32_t b = b0 + j * kThreads + tid;
            if (b >= c.to)
                continue;
            float x[N];
            uint32_t there;
            columns_of<T, Mask>(c, b, block[j], x, there);
            any |= there;
            const float most = largest_of(x);
            // (the line may be one of this list's own numbers, of a later tile than one that equals it: the equal ones go in as well)
            if (most >= line && most > -INFINITY)
                put(s, c, b, x, line, true);
            add(sums, x, scale, most);
        }
    }
    if (Mask && any)
        s.allowed = 1;
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
        sums = join(sums, Sums<float>{__shfl_xor_sync(~0u, sums.shift, d), __shfl_xor_sync(~0u, sums.w, d), __shfl_xor_sync(~0u, sums.wd, d)});
    if (lane == 0)
        s.warp[tid / 32u] = sums;
    __syncthreads();
    uint32_t n = s.n;
    if (n > kListCap) { // read again, piece by piece, with the best of what came before
        uint32_t have = 0;
        line = -INFINITY;
        __syncthreads();
        for (uint32_t b0 = c.from; b0 < c.to; b0 += kThreads) {
            if (tid == 0)
                s.n = have;
            __syncthreads();
            const uint32_t b = b0 + tid;
            if (b < c.to) {
                Block<T> block;
                block.raw = c.base[b];
                float x[N];
                uint32_t there;
                columns_of<T, Mask>(c, b, block, x, there);
                put(s, c, b, x, line, false); // an equal one comes behind k that are as large
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
                    if (lane == 0)
                        s.line = least;
                }
                __syncthreads();
                line = s.line;
            }
        }
        n = have;
        __syncthreads();
    }
    rank_best(s, n, k);
    {
        const float most = s.n_best ? key_x(s.best[0]) : 0.0f;
        if (!greedy && most != INFINITY && fabsf(most * scale) == INFINITY) { // a row of the type's lowest value, as masks write it: again, x - most first
            float w = 0.0f, wd = 0.0f;
            for (uint32_t b = c.from + tid; b < c.to; b += kThreads) {
                Block<T> block;
                block.raw = c.base[b];
                float x[N];
                uint32_t there;
                columns_of<T, Mask>(c, b, block, x, there);
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    const float d = fmaxf((x[i] - most) * scale, kLeast), e = ex2_approx(d);
                    w += e;
                    wd += e * d;
                }
            }
#pragma unroll
            for (uint32_t d = 16; d; d >>= 1) {
                w += __shfl_xor_sync(~0u, w, d);
                wd += __shfl_xor_sync(~0u, wd, d);
            }
            if (lane == 0)
                s.warp[tid / 32u] = Sums<float>{0.0f, w, wd};
            __syncthreads();
            if (tid == 0) {
                Sums<float> all = s.warp[0];
                for (uint32_t i = 1; i < kWarps; ++i)
                    all = join(all, s.warp[i]);
                s.sums = Sums<double>{(double)most * (double)scale, all.w, all.wd};
            }
        } else if (tid == 0) {
            Sums<float> all = s.warp[0];
            for (uint32_t i = 1; i < kWarps; ++i)
                all = join(all, s.warp[i]);
            s.sums = Sums<double>{(double)all.shift, all.w, all.wd};
        }
    }
    if (slices > 1) {
        cluster.sync();
        if (slice == 0) {
            uint32_t total = 0;
            for (uint32_t g = 0; g < slices; ++g) { // every slice's best, one behind the other
                const Shared* other = cluster.map_shared_rank(&s, g);
                const uint32_t has = other->n_best;
                if (tid < has)
                    s.list[total + tid] = other->best[tid];
                total += has;
            }
            Sums<double> all = s.sums;
            uint32_t allowed = s.allowed;
            for (uint32_t g = 1; g < slices; ++g) {
                const Shared* other = cluster.map_shared_rank(&s, g);
                all = join(all, other->sums);
                allowed |= other->allowed;
            }
            __syncthreads();
            if (tid == 0) {
                s.sums = all;
                s.allowed = allowed;
            }
            rank_best(s, total, k);
        }
        cluster.sync();
        if (slice)
            return;
    }
    __syncthreads();
    const Sums<double> all = s.sums;
    const uint32_t n_best = s.n_best;
    const float most = n_best ? key_x(s.best[0]) : -INFINITY;
    // one token alone: greedy, an infinite logit, or logits that are so far from one another that none but the largest weighs anything
    const bool one = n_best && (greedy || most == INFINITY || !(all.w > 0.0f));
    const float log2_sum = one ? 0.0f : log2f(all.w);
    constexpr float ln2 = 0.693147180559945309417f;
    const double ahead = one || n_best == 0 ? 0.0 : (double)most * (double)scale - all.shift; // of the shift: what rounding it left
    auto logprob = [&](float x, uint32_t id) {
        if (n_best == 0 || !(x > -INFINITY)) // (NaN too)
            return -INFINITY;
        if (one)
            return id == key_id(s.best[0]) ? 0.0f : -INFINITY;
        return (float)(((double)x - (double)most) / (double)t + 0.693147180559945309417 * (ahead - (double)log2_sum));
    };
    if (o.logprob)
        for (uint32_t i = tid; i < r.n_given; i += kThreads) {
            const uint32_t id = (uint32_t)r.tokens[(size_t)row * r.n_given + i];
            float y = 0.0f; // of no token
            if (id < r.n_vocab) {
                const bool there = !Mask || (__ldg(c.mask + id / 32u) >> (id & 31u)) & 1u;
                float x;
                if constexpr (sizeof(T) == 4)
                    x = x0[id];
                else if constexpr (std::is_same<T, __half>::value)
                    x = __half2float(x0[id]);
                else
                    x = __bfloat162float(x0[id]);
                y = logprob(there ? x : -INFINITY, id);
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
            o.flags[row] = n_best ? 0u : MK_FLAG_NO_CANDIDATE | (Mask && !s.allowed ? MK_FLAG_ALL_MASKED : 0u);
    }
}

template <typename T, bool Mask>
cudaError_t launch(const mk_logprob_rows& r, const LogprobOut& o, cudaStream_t stream)
{
    uint32_t slices = 1;
    while (slices < kMaxCluster && r.rows * slices < 148u * 2u && r.n_vocab / (2u * slices) >= 2048u)
        slices *= 2u;
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
