// The C ABI of the sampling operators (include/consumer_int8_drafts.h): argument validation, then
// the launch. Pure host code up to the launch.
#include "consumer_int8_drafts.h"

#include "abi_checks.h"
#include "attention_plan.h"
#include "sampling_launch.h"
#include "sampling_plan.h"

namespace {

using ci8::abi_fail;
using ci8::abi_launched;
using ci8::aligned;
using ci8::as_stream;
using ci8::overlap;

static_assert(CI8_SAMPLING_WORKSPACE_BYTES == ci8::kSamplingWorkspaceBytes);

constexpr int64_t kMaxExtent = int64_t(1) << 46;  // bytes; far past any buffer of a GPU
using i128 = __int128;

struct Buffer {
  const void* p;
  int64_t bytes;
};
template <int kOutputs, int kInputs>
bool shared(const Buffer (&outputs)[kOutputs], const Buffer (&inputs)[kInputs]) {
  for (int i = 0; i < kOutputs; ++i) {
    for (const Buffer& in : inputs)
      if (in.p && overlap(outputs[i].p, outputs[i].bytes, in.p, in.bytes)) return true;
    for (int j = 0; j < i; ++j)
      if (overlap(outputs[i].p, outputs[i].bytes, outputs[j].p, outputs[j].bytes)) return true;
  }
  return false;
}

int check_rows(int64_t tokens, int64_t vocab) {
  if (!(tokens >= 0 && vocab >= 1))
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid rows: expected a vocabulary of 1 token or more");
  if (tokens > (1 << 24) || vocab > ci8::kMostVocab)
    return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
  return CI8_OK;
}

// Bytes of [tokens, vocab] with rows `stride` values apart; -1 if over kMaxExtent.
int64_t extent(int64_t tokens, int64_t vocab, int64_t stride, int64_t size) {
  if (tokens == 0) return 0;
  const i128 bytes = (i128(tokens - 1) * stride + vocab) * size;
  return bytes > kMaxExtent ? -1 : int64_t(bytes);
}

int check_matrix(const void* p, int64_t tokens, int64_t vocab, int64_t stride, int64_t size) {
  if (tokens > 1 && stride < vocab)
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid rows: they must not overlap");
  if (tokens > 0 && !p) return abi_fail(CI8_ERR_GEOMETRY, "Missing rows");
  if (!aligned(p, size)) return abi_fail(CI8_ERR_ALIGNMENT, "Rows require aligned values");
  if (extent(tokens, vocab, stride, size) < 0) return abi_fail(CI8_ERR_TOO_LARGE, "Rows too large");
  return CI8_OK;
}

}  // namespace

extern "C" {

int ci8_token_probs(const void* logits, int64_t logit_bits, int64_t logit_stride,
                    const float* temperature, float* probs, int64_t prob_stride, int64_t tokens,
                    int64_t vocab, void* workspace, void* stream) {
  if (int s = check_rows(tokens, vocab)) return s;
  if (logit_bits != 16 && logit_bits != 32)
    return abi_fail(CI8_ERR_GEOMETRY, "Logits are BF16 (16) or FP32 (32)");
  const int64_t size = logit_bits / 8;
  if (int s = check_matrix(logits, tokens, vocab, logit_stride, size)) return s;
  if (int s = check_matrix(probs, tokens, vocab, prob_stride, 4)) return s;
  if (!aligned(temperature, 4) || !aligned(workspace, 16) || !workspace)
    return abi_fail(CI8_ERR_ALIGNMENT, "token_probs requires aligned buffers");
  if (!ci8::launch_fits(tokens, ci8::kRowThreads))
    return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
  const int64_t in = extent(tokens, vocab, logit_stride, size);
  const int64_t out = extent(tokens, vocab, prob_stride, 4);
  const bool in_place = size == 4 && logits == probs && (logit_stride == prob_stride || tokens <= 1);
  const Buffer outputs[] = {{probs, out}, {workspace, ci8::kSamplingWorkspaceBytes}};
  const Buffer inputs[] = {{temperature, tokens * 4}};
  if (shared(outputs, inputs) || (!in_place && overlap(probs, out, logits, in)) ||
      overlap(workspace, ci8::kSamplingWorkspaceBytes, logits, in))
    return abi_fail(CI8_ERR_OVERLAP, "token_probs outputs must not overlap anything else");
  ci8::ProbsArgs args = {};
  args.logits = logits;
  args.temperature = temperature;
  args.probs = probs;
  args.workspace = static_cast<float*>(workspace);
  args.logit_stride = logit_stride;
  args.prob_stride = prob_stride;
  args.tokens = int(tokens);
  args.vocab = int(vocab);
  return abi_launched(ci8::launch_token_probs(args, logit_bits == 16, as_stream(stream)));
}

int ci8_verify_drafts(const float* target, int64_t target_stride, const float* draft,
                      int64_t draft_stride, const int64_t* ids, const int32_t* parents,
                      const int32_t* q_starts, const float* uniforms, int64_t seqs, int64_t tokens,
                      int64_t vocab, void* workspace, int32_t* path, int32_t* accepted,
                      int64_t* next, void* stream) {
  if (int s = check_rows(tokens, vocab)) return s;
  if (!(seqs >= 0 && seqs <= ci8::kMostVerified))
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid verification: expected at most 16384 sequences");
  if (int s = check_matrix(target, tokens, vocab, target_stride, 4)) return s;
  if (draft)
    if (int s = check_matrix(draft, tokens, vocab, draft_stride, 4)) return s;
  if ((seqs > 0 && (!q_starts || !accepted || !next)) ||
      (seqs > 0 && tokens > 0 && (!ids || !uniforms || !path)))
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid verification: a buffer is missing");
  if (!aligned(ids, 8) || !aligned(parents, 4) || !aligned(q_starts, 4) || !aligned(uniforms, 4) ||
      !aligned(workspace, 16) || !workspace || !aligned(path, 4) || !aligned(accepted, 4) ||
      !aligned(next, 8))
    return abi_fail(CI8_ERR_ALIGNMENT, "verify_drafts requires aligned buffers");
  const Buffer outputs[] = {{path, tokens * 4},
                            {accepted, seqs * 4},
                            {next, seqs * 8},
                            {workspace, ci8::kSamplingWorkspaceBytes}};
  const Buffer inputs[] = {{target, extent(tokens, vocab, target_stride, 4)},
                           {draft, draft ? extent(tokens, vocab, draft_stride, 4) : 0},
                           {ids, tokens * 8},
                           {parents, tokens * 4},
                           {q_starts, (seqs + 1) * 4},
                           {uniforms, tokens * 4}};
  if (shared(outputs, inputs))
    return abi_fail(CI8_ERR_OVERLAP, "verify_drafts outputs must not overlap anything else");
  ci8::VerifyArgs args = {};
  args.target = target;
  args.draft = draft;
  args.ids = ids;
  args.parents = parents;
  args.q_starts = q_starts;
  args.uniforms = uniforms;
  args.workspace = workspace;
  args.path = path;
  args.accepted = accepted;
  args.next = next;
  args.target_stride = target_stride;
  args.draft_stride = draft_stride;
  args.seqs = int(seqs);
  args.tokens = int(tokens);
  args.vocab = int(vocab);
  return abi_launched(ci8::launch_verify_drafts(args, as_stream(stream)));
}

}  // extern "C"
