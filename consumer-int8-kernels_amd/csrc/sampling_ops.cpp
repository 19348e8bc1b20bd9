// torch.ops.consumer_int8 registration of the sampling operators over their C ABI
// (include/consumer_int8_drafts.h), as in attention_ops.cpp.
#include "consumer_int8_drafts.h"
#include "torch_checks.h"

namespace {

// [tokens, vocab] with contiguous values: how far apart its rows are. The stride of an axis of length
// 1 says nothing.
int64_t row_stride(const Tensor& t) {
  STD_TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1),
                  "Expected rows [tokens, vocab] with contiguous values");
  return t.size(0) <= 1 ? t.size(1) : t.stride(0);
}

void check_vector(const Tensor& t, ScalarType dtype, int64_t length, int device) {
  check_plain(t, dtype, device);
  STD_TORCH_CHECK(t.dim() == 1 && t.size(0) == length, "Unexpected length of a vector");
}

void check_workspace(const Tensor& t, int device) {
  check_plain(t, ScalarType::Float, device);
  STD_TORCH_CHECK(t.numel() * 4 >= CI8_SAMPLING_WORKSPACE_BYTES, "Expected an FP32 workspace [262144]");
}

void token_probs(Tensor logits, MaybeTensor temperature, Tensor workspace, Tensor probs) {
  const int device = logits.get_device_index();
  const bool bf16 = logits.scalar_type() == ScalarType::BFloat16;
  check_type(logits, bf16 ? ScalarType::BFloat16 : ScalarType::Float, device);
  check_type(probs, ScalarType::Float, device);
  const int64_t logit_stride = row_stride(logits), prob_stride = row_stride(probs);
  const int64_t tokens = logits.size(0), vocab = logits.size(1);
  STD_TORCH_CHECK(probs.size(0) == tokens && probs.size(1) == vocab,
                  "Probabilities must have the logits' shape");
  if (temperature.has_value()) check_vector(*temperature, ScalarType::Float, tokens, device);
  check_workspace(workspace, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_token_probs(
      logits.data_ptr(), bf16 ? 16 : 32, logit_stride,
      temperature.has_value() ? static_cast<const float*>(temperature->data_ptr()) : nullptr,
      static_cast<float*>(probs.data_ptr()), prob_stride, tokens, vocab, workspace.data_ptr(),
      stream_for(device)));
}

void verify_drafts(Tensor target, MaybeTensor draft, Tensor tokens, MaybeTensor parents,
                   Tensor q_starts, Tensor uniforms, Tensor workspace, Tensor path, Tensor accepted,
                   Tensor next) {
  const int device = target.get_device_index();
  check_type(target, ScalarType::Float, device);
  const int64_t target_stride = row_stride(target);
  const int64_t rows = target.size(0), vocab = target.size(1);
  int64_t draft_stride = 0;
  if (draft.has_value()) {
    check_type(*draft, ScalarType::Float, device);
    draft_stride = row_stride(*draft);
    STD_TORCH_CHECK(draft->size(0) == rows && draft->size(1) == vocab,
                    "Draft probabilities must have the target's shape");
  }
  check_vector(tokens, ScalarType::Long, rows, device);
  if (parents.has_value()) check_vector(*parents, ScalarType::Int, rows, device);
  check_vector(uniforms, ScalarType::Float, rows, device);
  check_vector(path, ScalarType::Int, rows, device);
  check_plain(q_starts, ScalarType::Int, device);
  STD_TORCH_CHECK(q_starts.dim() == 1 && q_starts.size(0) >= 1,
                  "Expected INT32 q_starts [seqs + 1]");
  const int64_t seqs = q_starts.size(0) - 1;
  check_vector(accepted, ScalarType::Int, seqs, device);
  check_vector(next, ScalarType::Long, seqs, device);
  check_workspace(workspace, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_verify_drafts(
      static_cast<const float*>(target.data_ptr()), target_stride,
      draft.has_value() ? static_cast<const float*>(draft->data_ptr()) : nullptr, draft_stride,
      static_cast<const int64_t*>(tokens.data_ptr()),
      parents.has_value() ? static_cast<const int32_t*>(parents->data_ptr()) : nullptr,
      static_cast<const int32_t*>(q_starts.data_ptr()),
      static_cast<const float*>(uniforms.data_ptr()), seqs, rows, vocab, workspace.data_ptr(),
      static_cast<int32_t*>(path.data_ptr()), static_cast<int32_t*>(accepted.data_ptr()),
      static_cast<int64_t*>(next.data_ptr()), stream_for(device)));
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(consumer_int8, m) {
  m.def("token_probs(Tensor logits, Tensor? temperature, Tensor(a!) workspace, Tensor(b!) probs) -> ()");
  m.def("verify_drafts(Tensor target_probs, Tensor? draft_probs, Tensor tokens, Tensor? parents, Tensor q_starts, Tensor uniforms, Tensor(a!) workspace, Tensor(b!) path, Tensor(c!) accepted, Tensor(d!) next_tokens) -> ()");
}

STABLE_TORCH_LIBRARY_IMPL(consumer_int8, CUDA, m) {
  m.impl("token_probs", TORCH_BOX(&token_probs));
  m.impl("verify_drafts", TORCH_BOX(&verify_drafts));
}
