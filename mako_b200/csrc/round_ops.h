// Host-visible declarations of the operators of a serving round around the sampler (internal to the library; the public
// surface is include/mako_b200.h): the head with adapters, the verification of drafts against distributions, the page plan.
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

} // namespace mk
