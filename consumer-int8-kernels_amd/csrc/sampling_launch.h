// Internal host launchers of the sampling operators, called by the validated C ABI in
// sampling_abi.cpp. Arguments are assumed valid; each returns the launch status.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace ci8 {

struct ProbsArgs {
  const void* logits;
  const float* temperature;  // null: 1
  float* probs;
  float* workspace;
  int64_t logit_stride, prob_stride;
  int tokens, vocab;
};
hipError_t launch_token_probs(const ProbsArgs& args, bool bf16, hipStream_t stream);

struct VerifyArgs {
  const float* target;
  const float* draft;  // null: drafts are certain choices
  const int64_t* ids;
  const int32_t* parents;  // null: chains
  const int32_t* q_starts;
  const float* uniforms;
  void* workspace;
  int32_t* path;
  int32_t* accepted;
  int64_t* next;
  int64_t target_stride, draft_stride;
  int seqs, tokens, vocab;
};
hipError_t launch_verify_drafts(const VerifyArgs& args, hipStream_t stream);

}  // namespace ci8
