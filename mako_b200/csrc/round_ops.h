// Host-visible declarations of the operators of a serving round around the sampler (internal to the library; the public
// surface is include/mako_b200.h): the head with adapters, the verification of drafts against distributions, the page plan.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/mako_b200.h"

namespace mk {

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

struct SpecVerifyArgs {
    mk_spec_rows r;
    int32_t *n_kept, *next_token, *tokens;
    float* logprob;
    uint32_t* flags;
};
cudaError_t launch_spec_verify(const SpecVerifyArgs& a, cudaStream_t stream);

struct KvPlanArgs {
    mk_kv_pages p;
    mk_kv_plan o;
    const int32_t *cache_len, *n_new;
    uint32_t n_seq;
};
cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t stream);

} // namespace mk
