// For tests, in the measurement library: verify_drafts whose workgroups look for each other's sums not
// once, so that each adds up all chunks itself, as after a wait in vain.
#define CI8_MOST_POLLS 0
#define launch_token_probs probe_launch_token_probs
#define launch_verify_drafts probe_launch_verify_drafts
#include "sampling.hip"

extern "C" int probe_verify_drafts(const float* target, const float* draft, const int64_t* ids,
                                   const int32_t* parents, const int32_t* q_starts,
                                   const float* uniforms, int64_t seqs, int64_t tokens, int64_t vocab,
                                   void* workspace, int32_t* path, int32_t* accepted, int64_t* next,
                                   void* stream) {
  if (seqs < 1 || seqs > ci8::kMostVerified || tokens < 1 || tokens > (1 << 24) || vocab < 1 ||
      vocab > ci8::kMostVocab)
    return int(hipErrorInvalidValue);
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
  args.target_stride = args.draft_stride = vocab;
  args.seqs = int(seqs);
  args.tokens = int(tokens);
  args.vocab = int(vocab);
  return int(ci8::probe_launch_verify_drafts(args, static_cast<hipStream_t>(stream)));
}
