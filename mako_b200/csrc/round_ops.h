// Host-visible declarations of the operators of a serving round around the sampler (internal to the library; the public
// surface is include/mako_b200.h): the head with adapters, the verification of drafts against distributions, the page plan, the
// cache behind it, the log-probabilities of tokens.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/mako_b200.h"

namespace mk {

// Sets a kernel's attribute, once on each of the first 64 devices: a call takes about a microsecond. `done`: the kernel's own.
template <typename K>
cudaError_t set_once(std::atomic<uint64_t>& done, K* kernel, cudaFuncAttribute attr, int value)
{
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && (done.load(std::memory_order_relaxed) >> device & 1u)))
        return e;
    e = cudaFuncSetAttribute(kernel, attr, value);
    if (e == cudaSuccess && device < 64)
        done.fetch_or(1ull << device, std::memory_order_relaxed);
    return e;
}

constexpr uint32_t kHeadMaxRank = 128;
// What a call with adapters needs of the handle, for its rows: `hidden` [rows][dim] of the matrices' type on a 16-byte boundary,
// `ints` [2][rows], `inner` [rows][kHeadMaxRank].
struct HeadScratch {
    void* hidden;
    int32_t* ints;
    float* inner;
};
cudaError_t launch_head_logits(const mk_head& h, const void* hidden, uint64_t hidden_ld, const int32_t* adapter, uint32_t rows,
                               const HeadScratch& scratch, float* logits, uint64_t ld, cudaStream_t stream);

// What a slice of a position's rows leaves, and what becomes of the position: maximum and sum of the target's and the drafter's
// row, the first column that holds the maximum (where that matters).
struct SpecPart {
    float m_p, s_p;
    uint32_t at_p, unused_p;
    float m_q, s_q;
    uint32_t at_q, unused_q;
};
struct SpecState {
    float m_p, s_p;
    uint32_t at_p, state;
    float m_q, s_q;
    uint32_t at_q, unused;
};
constexpr uint32_t kSpecPositions = 33; // words of counters a row of a handle has: 32 positions and the round's end
inline uint32_t spec_slices(uint32_t n_vocab) { return n_vocab / 1024u + 1u < 64u ? n_vocab / 1024u + 1u : 64u; }

struct SpecVerifyArgs {
    mk_spec_rows r;
    int32_t *n_kept, *next_token, *tokens;
    float* logprob;
    uint32_t* flags;
    // the handle's: [n_seq * n_pos][slices], [n_seq * n_pos], and counters that are zero between calls: [n_seq * n_pos], [n_seq], one
    // of the work taken, and one that stays up once a wait has run out
    SpecPart* parts;
    SpecState* states;
    uint32_t *tickets, *ended, *counter, *failed;
    uint32_t slices; // at most
};
cudaError_t launch_spec_verify(const SpecVerifyArgs& a, cudaStream_t stream);

constexpr uint32_t kPlanMaxSeq = 8192;
struct KvPlanArgs {
    mk_kv_pages p;
    mk_kv_plan o;
    const int32_t *cache_len, *n_new;
    uint32_t n_seq;
};
cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t stream);

constexpr uint32_t kLogprobMaxTop = 64;
struct LogprobOut {
    float *logprob, *entropy;
    int32_t* top_ids;
    float* top_logprob;
    uint32_t* flags;
};
cudaError_t launch_token_logprobs(const mk_logprob_rows& r, const LogprobOut& o, cudaStream_t stream);

constexpr uint32_t kAppendMaxGroup = 8192; // query heads of a key head: 65536 tokens' rows of two key heads are counted in 31 bits
struct KvAppendArgs {
    mk_kv_cache c;
    const void *q, *k, *v;
    void* q_out;
    uint64_t q_ld, k_ld, v_ld, q_out_ld;
    const int32_t* positions;
    const int64_t* slots;
    uint32_t n_tokens, group; // query heads of a key head; 0: no queries
    const float* inv_freq;
    uint32_t rotary;          // columns that turn, or 0
    bool interleaved;
    float rotary_scale;
    uint32_t tokens_each;     // of a CTA; the launch sets it
};
cudaError_t launch_kv_append(const KvAppendArgs& a, int type, cudaStream_t stream);

struct KvAttendArgs {
    mk_kv_cache c;
    const void* q;
    void* out;
    uint64_t q_ld, out_ld;
    const int32_t* block_table;
    uint64_t table_ld;
    const int32_t *query_start, *kv_len;
    float* parts;
    uint64_t page_inverse, group_inverse;
    uint32_t page_shift, group_shift, table_cols, n_seq, n_tokens, max_new, group, window;
    float scale_log2;         // of a score, for exponents of two
    // which sequences a launch takes, by their rows (tokens of the pass times group), the least blocks of a CTA, and how many of them a unit
    // costs beside its own; the launch sets them
    uint32_t rows_from, rows_to, blocks_least, unit_cost;
};
constexpr uint32_t kPromptCtas = 148, kPromptRows = 256, kPromptBlock = 128; // CTAs; rows of a unit; keys of a block
uint64_t kv_attend_bytes(uint32_t dim, uint64_t most_rows); // of parts; rows: of a sequence
cudaError_t launch_kv_prompt(const KvAttendArgs& a, int type, cudaStream_t stream);
cudaError_t launch_kv_attend(const KvAttendArgs& a, int type, cudaStream_t stream);

} // namespace mk
