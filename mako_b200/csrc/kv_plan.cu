// Block tables and slot maps of a paged cache from the sequences' lengths (mk_kv_plan_step in include/mako_b200.h). All of it is
// running sums over the sequences: of the tokens (which of them fit), of the pages given back, of the pages taken, of the tokens
// of those that run. One CTA; a thread per sequence, 1024 at a time, with the sums carried from one thousand to the next.
#include "round_ops.h"

namespace mk {
namespace {

constexpr uint32_t kPlanThreads = 1024;

struct Scan {
    long long warp[32];
};

// Inclusive running sum over the CTA, `total` of all. Every thread calls it.
__device__ long long block_scan(Scan& s, long long x, long long& total)
{
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(~0u, x, d);
        x += lane >= d ? y : 0;
    }
    __syncthreads(); // the sums of the call before have been read
    if (lane == 31)
        s.warp[w] = x;
    __syncthreads();
    long long before = 0, all = 0;
    for (uint32_t i = 0; i < kPlanThreads / 32; ++i) {
        const long long v = s.warp[i];
        before += i < w ? v : 0;
        all += v;
    }
    total = all;
    return x + before;
}

struct Seq {
    long long len, fresh, held, want;
    bool bad, over;
};

__device__ Seq read_seq(const KvPlanArgs& a, uint32_t s)
{
    Seq q{0, 0, 0, 0, true, false};
    if (s >= a.n_seq)
        return q;
    q.len = a.cache_len[s];
    q.fresh = a.n_new ? a.n_new[s] : 0;
    q.held = a.p.n_pages[s];
    const long long end = q.len + q.fresh;
    q.want = (end + a.p.page_size - 1) / a.p.page_size;
    q.bad = q.len < 0 || q.fresh < 0 || q.held < 0 || q.held > a.p.table_cols || q.want > a.p.table_cols || end > 0x7fffffffll;
    return q;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const KvPlanArgs a)
{
    __shared__ Scan s_scan;
    const uint32_t tid = threadIdx.x;
    const long long cap = a.p.free_cap;
    long long n_free = *a.p.n_free;
    n_free = n_free < 0 ? 0 : n_free > cap ? cap : n_free;
    long long given = 0, total, tokens = 0;
    for (uint32_t base = 0; base < a.n_seq; base += kPlanThreads) { // how many pages come back
        Seq q = read_seq(a, base + tid);
        const long long upto = tokens + block_scan(s_scan, q.bad ? 0 : q.fresh, total);
        tokens += total;
        q.over = !q.bad && q.fresh > 0 && upto > a.o.max_tokens;
        block_scan(s_scan, !q.bad && !q.over && q.held > q.want ? q.held - q.want : 0, total);
        given += total;
    }
    if (n_free + given > cap)
        given = 0;
    const long long top = n_free + given;
    long long back = 0;
    tokens = 0;
    if (given)
        for (uint32_t base = 0; base < a.n_seq; base += kPlanThreads) {
            Seq q = read_seq(a, base + tid);
            const long long upto = tokens + block_scan(s_scan, q.bad ? 0 : q.fresh, total);
            tokens += total;
            q.over = !q.bad && q.fresh > 0 && upto > a.o.max_tokens;
            const long long give = !q.bad && !q.over && q.held > q.want ? q.held - q.want : 0;
            const long long rank = back + block_scan(s_scan, give, total) - give;
            back += total;
            for (long long i = 0; i < give; ++i) {
                int32_t* e = a.p.block_table + (size_t)(base + tid) * a.p.table_ld + q.want + i;
                a.p.free_list[top - 1 - rank - i] = *e;
                *e = -1;
            }
        }
    __syncthreads(); // the list is whole before pages are taken from it
    long long taken = 0, granted = 0, start = 0;
    tokens = 0;
    for (uint32_t base = 0; base < a.n_seq; base += kPlanThreads) {
        const uint32_t s = base + tid;
        Seq q = read_seq(a, s);
        const long long upto = tokens + block_scan(s_scan, q.bad ? 0 : q.fresh, total);
        tokens += total;
        q.over = !q.bad && q.fresh > 0 && upto > a.o.max_tokens;
        const bool part = !q.bad && !q.over;
        const long long take = part && q.want > q.held ? q.want - q.held : 0;
        const long long rank = taken + block_scan(s_scan, take, total) - take;
        taken += total;
        const bool lack = take > 0 && rank + take > top;
        block_scan(s_scan, lack ? 0 : take, total);
        granted += total;
        const long long run = part && !lack ? q.fresh : 0;
        const long long first = start + block_scan(s_scan, run, total) - run;
        start += total;
        if (s < a.n_seq) {
            int32_t* row = a.p.block_table + (size_t)s * a.p.table_ld;
            for (long long i = 0; i < take && !lack; ++i)
                row[q.held + i] = a.p.free_list[top - 1 - rank - i];
            if (part && !lack)
                a.p.n_pages[s] = (int32_t)(q.held > q.want && !given ? q.held : q.want);
            if (a.o.query_start)
                a.o.query_start[s] = (int32_t)first;
            if (a.o.kv_len)
                a.o.kv_len[s] = q.bad ? 0 : (int32_t)(q.len + run);
            if (a.o.flags)
                a.o.flags[s] = q.bad ? MK_FLAG_PLAN_INVALID : q.over ? MK_FLAG_NO_ROOM : lack ? MK_FLAG_NO_PAGES : 0u;
            for (long long i = 0; i < run; ++i) {
                const long long at = q.len + i;
                if (a.o.positions)
                    a.o.positions[first + i] = (int32_t)at;
                if (a.o.slots)
                    a.o.slots[first + i] = (long long)row[at / a.p.page_size] * a.p.page_size + at % a.p.page_size;
                if (a.o.token_seq)
                    a.o.token_seq[first + i] = (int32_t)s;
            }
        }
    }
    if (tid == 0) {
        *a.p.n_free = (int32_t)(top - granted);
        if (a.o.query_start)
            a.o.query_start[a.n_seq] = (int32_t)start;
    }
    for (long long t = start + tid; t < a.o.max_tokens; t += kPlanThreads) {
        if (a.o.positions)
            a.o.positions[t] = 0;
        if (a.o.slots)
            a.o.slots[t] = -1;
        if (a.o.token_seq)
            a.o.token_seq[t] = -1;
    }
}

} // namespace

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t stream)
{
    kv_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

} // namespace mk
