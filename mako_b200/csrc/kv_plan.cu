// Block tables and slot maps of a paged cache from the sequences' lengths (mk_kv_plan_step in include/mako_b200.h). A few kilobytes go
// in and out: what bounds it is latency, of the launch and of a chain of reads, sums and look-ups. 5.5 us for 256 sequences, 7 for
// 1000 with 8000 rows in two launches, in a graph.
//
// One CTA plans. A thread has a run of sequences (one each up to 1024), and a single pass of running sums gives where the tokens
// of each start and which pages of the list are whose; tokens and pages are then dealt out to the threads evenly, each finding its
// sequence by bisection, so that neither a long prompt nor a sequence that gives back a thousand pages is one thread's work. The sums
// assume that all sequences fit; where a total says otherwise they are formed again without those that do not. Up to kPlanTokens
// rows the same CTA writes them, more are written by a second launch of as many CTAs as there is work for.
#include "ptx.cuh"
#include "round_ops.h"

namespace mk {
namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanTokens = 4096, kTokenThreads = 256;
constexpr uint32_t kSeqBytes = 3 * 4; // of shared memory: three running sums

struct Sums {
    long long tokens, give, take;
    __device__ Sums operator+(const Sums& o) const { return Sums{tokens + o.tokens, give + o.give, take + o.take}; }
};

struct Shared {
    Sums warp[kPlanWarps];
    long long n_free;
};

__device__ __forceinline__ Sums before_in_warp(Sums x) // of the lanes in front, by running sums
{
    const uint32_t lane = threadIdx.x & 31u;
    Sums run = x;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const Sums y{__shfl_up_sync(~0u, run.tokens, d), __shfl_up_sync(~0u, run.give, d), __shfl_up_sync(~0u, run.take, d)};
        if (lane >= d)
            run = run + y;
    }
    return Sums{run.tokens - x.tokens, run.give - x.give, run.take - x.take};
}

// The sum of all threads' x in front of this one, and of all.
__device__ Sums before_in_cta(Shared& s, const Sums& x, Sums& total)
{
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x / 32u;
    const Sums before = before_in_warp(x);
    __syncthreads(); // the sums before these have been read
    if (lane == 31u)
        s.warp[w] = before + x;
    __syncthreads();
    const Sums of = s.warp[lane], front = before_in_warp(of), all = front + of;
    total = Sums{__shfl_sync(~0u, all.tokens, 31), __shfl_sync(~0u, all.give, 31), __shfl_sync(~0u, all.take, 31)};
    return before + Sums{__shfl_sync(~0u, front.tokens, w), __shfl_sync(~0u, front.give, w), __shfl_sync(~0u, front.take, w)};
}

struct Seq {
    long long len, fresh, held, want;
    bool bad;
};

__device__ __forceinline__ Seq read_seq(const KvPlanArgs& a, uint32_t s)
{
    Seq q;
    q.len = a.cache_len[s];
    q.fresh = a.n_new ? a.n_new[s] : 0;
    q.held = a.p.n_pages[s];
    const long long end = q.len + q.fresh;
    q.bad = q.len < 0 || q.fresh < 0 || q.held < 0 || q.held > a.p.table_cols || end > 0x7fffffffll;
    q.want = q.bad ? 0 : ((uint32_t)end + (a.p.page_size - 1ull)) / a.p.page_size;
    q.bad = q.bad || q.want > a.p.table_cols;
    return q;
}

// The last place in [0, n) whose number, of an ascending array that starts with 0, is at most i.
__device__ __forceinline__ uint32_t last_at_most(const uint32_t* a, uint32_t n, uint32_t i)
{
    uint32_t low = 0;
    for (uint32_t step = 1u << (31 - __clz((int)n)); step; step >>= 1)
        if (low + step < n && a[low + step] <= i)
            low += step;
    return low;
}

// One row of the pass, or of the padding behind it.
__device__ __forceinline__ void write_token(const KvPlanArgs& a, const uint32_t* start, uint32_t total, uint32_t t)
{
    uint32_t at = 0;
    int32_t seq = -1;
    long long slot = -1;
    if (t < total) {
        const uint32_t s = last_at_most(start, a.n_seq, t);
        at = (uint32_t)a.cache_len[s] + (t - start[s]);
        const uint32_t page = at / a.p.page_size;
        seq = (int32_t)s;
        if (a.o.slots)
            slot = (long long)a.p.block_table[(size_t)s * a.p.table_ld + page] * a.p.page_size + (at - page * a.p.page_size);
    }
    if (a.o.positions)
        a.o.positions[t] = (int32_t)at;
    if (a.o.slots)
        a.o.slots[t] = slot;
    if (a.o.token_seq)
        a.o.token_seq[t] = seq;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const KvPlanArgs a, const bool with_tokens)
{
    extern __shared__ uint32_t arrays[]; // of each sequence: where its tokens, what it gives and what it takes start
    __shared__ Shared s;
    griddep_launch_dependents();
    uint32_t *start = arrays, *gives = start + a.n_seq, *takes = gives + a.n_seq;
    const uint32_t tid = threadIdx.x, each = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
    const uint32_t s0 = min(tid * each, a.n_seq), s1 = min(s0 + each, a.n_seq);
    const long long cap = a.p.free_cap, most = a.o.max_tokens;
    if (tid == 0) {
        const long long f = *a.p.n_free;
        s.n_free = f < 0 ? 0 : f > cap ? cap : f;
    }
    // what a sequence adds to the sums; upto: the tokens of valid ones up to its end
    auto of_seq = [&](const Seq& q, long long upto, bool& over) {
        over = !q.bad && q.fresh > 0 && upto > most;
        const bool part = !q.bad && !over;
        return Sums{q.bad ? 0 : q.fresh, part && q.held > q.want ? q.held - q.want : 0, part && q.want > q.held ? q.want - q.held : 0};
    };
    Sums mine{0, 0, 0}, total;
    Seq first{0, 0, 0, 0, true};
    bool over;
    for (uint32_t i = s0; i < s1; ++i) {
        const Seq q = read_seq(a, i);
        if (i == s0)
            first = q;
        mine = mine + of_seq(q, 0, over);
    }
    Sums at = before_in_cta(s, mine, total);
    if (total.tokens > most) { // once more, with what the tokens in front say
        const long long front = at.tokens;
        mine = Sums{0, 0, 0};
        for (uint32_t i = s0; i < s1; ++i) {
            const Seq q = i == s0 ? first : read_seq(a, i);
            mine = mine + of_seq(q, front + mine.tokens + (q.bad ? 0 : q.fresh), over);
        }
        at = before_in_cta(s, mine, total);
    }
    const bool room = s.n_free + total.give <= cap;
    const long long given = room ? total.give : 0, top = s.n_free + given;
    // which sequences run: where all do, their tokens start at the sums that are there already
    const bool all_run = total.tokens <= most && total.take <= top;
    long long begin = at.tokens, taken = total.take;
    if (!all_run) {
        Sums run{0, 0, 0}, all;
        Sums go = at;
        for (uint32_t i = s0; i < s1; ++i) {
            const Seq q = i == s0 ? first : read_seq(a, i);
            const Sums x = of_seq(q, go.tokens + (q.bad ? 0 : q.fresh), over);
            go = go + x;
            const bool lack = x.take > 0 && go.take > top;
            run = run + Sums{q.bad || over || lack ? 0 : q.fresh, 0, lack ? 0 : x.take};
        }
        begin = before_in_cta(s, run, all).tokens;
        total.tokens = all.tokens;
        taken = all.take;
    }
    Sums go = at;
    for (uint32_t i = s0; i < s1; ++i) {
        const Seq q = i == s0 ? first : read_seq(a, i);
        const Sums x = of_seq(q, go.tokens + (q.bad ? 0 : q.fresh), over);
        const bool lack = x.take > 0 && go.take + x.take > top, runs = !q.bad && !over && !lack;
        const long long fresh = runs ? q.fresh : 0;
        start[i] = (uint32_t)begin;
        gives[i] = (uint32_t)go.give;
        takes[i] = (uint32_t)(go.take < taken ? go.take : taken);
        if (a.o.query_start)
            a.o.query_start[i] = (int32_t)begin;
        if (a.o.kv_len)
            a.o.kv_len[i] = q.bad ? 0 : (int32_t)(q.len + fresh);
        if (a.o.flags)
            a.o.flags[i] = q.bad ? MK_FLAG_PLAN_INVALID : over ? MK_FLAG_NO_ROOM : lack ? MK_FLAG_NO_PAGES : 0u;
        begin += fresh;
        go = go + x;
    }
    if (tid == 0) {
        *a.p.n_free = (int32_t)(top - taken);
        if (a.o.query_start)
            a.o.query_start[a.n_seq] = (int32_t)total.tokens;
    }
    __syncthreads();
    // pages that come back go on top of the list, the first of them topmost
    for (uint32_t i = tid; i < (uint32_t)given; i += kPlanThreads) {
        const uint32_t q = last_at_most(gives, a.n_seq, i), next = q + 1u < a.n_seq ? gives[q + 1u] : (uint32_t)given;
        int32_t* e = a.p.block_table + (size_t)q * a.p.table_ld + (uint32_t)a.p.n_pages[q] - (next - i);
        a.p.free_list[top - 1 - i] = *e;
        *e = -1;
    }
    if (given)
        __syncthreads(); // the list is whole before pages are taken from it
    for (uint32_t i = tid; i < (uint32_t)taken; i += kPlanThreads) {
        const uint32_t q = last_at_most(takes, a.n_seq, i);
        a.p.block_table[(size_t)q * a.p.table_ld + (uint32_t)a.p.n_pages[q] + (i - takes[q])] = a.p.free_list[top - 1 - i];
    }
    __syncthreads(); // n_pages has been read
    for (uint32_t i = s0; i < s1; ++i) {
        const uint32_t give = (i + 1u < a.n_seq ? gives[i + 1u] : (uint32_t)total.give) - gives[i];
        const uint32_t take = (i + 1u < a.n_seq ? takes[i + 1u] : (uint32_t)taken) - takes[i];
        if ((give && room) || take)
            a.p.n_pages[i] = a.p.n_pages[i] - (int32_t)give + (int32_t)take;
    }
    if (with_tokens)
        for (uint32_t t = tid; t < a.o.max_tokens; t += kPlanThreads)
            write_token(a, start, (uint32_t)total.tokens, t);
}

// The rows of a larger pass, behind the plan.
__global__ void __launch_bounds__(kTokenThreads) kv_token_kernel(const KvPlanArgs a)
{
    extern __shared__ uint32_t start[];
    griddep_wait();
    for (uint32_t i = threadIdx.x; i <= a.n_seq; i += kTokenThreads)
        start[i] = (uint32_t)a.o.query_start[i];
    __syncthreads();
    for (uint32_t t = blockIdx.x * kTokenThreads + threadIdx.x; t < a.o.max_tokens; t += gridDim.x * kTokenThreads)
        write_token(a, start, start[a.n_seq], t);
}

} // namespace

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t stream)
{
    // What a call may ask for is set once, for the most sequences there are: it belongs to the kernel, not to the call, so that one
    // thread's call must not lower it under another's. (Without it dynamic and static shared memory have 48 KB together: 4030 sequences.)
    static std::atomic<uint64_t> room_set{0};
    const size_t smem = (size_t)a.n_seq * kSeqBytes;
    cudaError_t e = set_once(room_set, kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kPlanMaxSeq * kSeqBytes));
    if (e != cudaSuccess)
        return e;
    const bool rows = a.o.positions || a.o.slots || a.o.token_seq, here = a.o.max_tokens <= kPlanTokens;
    kv_plan_kernel<<<1, kPlanThreads, smem, stream>>>(a, rows && here);
    e = cudaGetLastError();
    if (e != cudaSuccess || !rows || here)
        return e;
    const uint32_t work = (a.o.max_tokens + kTokenThreads - 1) / kTokenThreads;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(work < 148u * 8u ? work : 148u * 8u);
    c.blockDim = dim3(kTokenThreads);
    c.dynamicSmemBytes = ((size_t)a.n_seq + 1u) * 4u;
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kv_token_kernel, a);
}

} // namespace mk
