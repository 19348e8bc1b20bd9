// Internal host launchers of the attention operators, called by the validated C ABI in
// attention_abi.cpp. Arguments are assumed valid; each returns the launch status.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace ci8 {

// BF16 heads (ci8_heads): element strides.
struct HeadsView {
  uint16_t* data;
  int heads;
  int64_t token_stride, head_stride;
};

// ci8_rotation; rot = 0 rotates nothing.
struct RotationView {
  const float* table;
  const int64_t* positions;
  const int32_t* axis_of;
  int64_t rows;
  int rot, axes;
  bool interleaved;
};

// Codes and scales of the keys or of the values: [pages, heads, page_size, .] bytes.
struct Fp4Rows {
  uint8_t* codes;
  uint8_t* scales;
  int64_t code_stride, scale_stride;  // bytes between pages
};
struct Fp4CacheView {
  Fp4Rows k, v;
  int pages, heads, page_shift;  // page_size = 1 << page_shift
};

struct NormRopeArgs {
  HeadsView q, k, v, q_out, k_out;  // v and slots: append only; q.heads = 0: no queries
  const float* q_weight;
  const float* k_weight;
  float eps;
  RotationView rotation;
  const int64_t* slots;
  Fp4CacheView cache;
  int tokens;
};
hipError_t launch_norm_rope(const NormRopeArgs& args, int dim, bool append, hipStream_t stream);

hipError_t launch_unpack_fp4(const Fp4CacheView& cache, const int64_t* slots, uint16_t* k,
                             uint16_t* v, int count, int dim, hipStream_t stream);

hipError_t launch_move_fp4(const Fp4CacheView& cache, const int32_t* rows, const int64_t* slots,
                           const int32_t* q_starts, int seqs, int tokens, int dim,
                           hipStream_t stream);

// Rows of partial sums that the workspace holds, FP32 [rows, dim] and then [rows, 2].
constexpr int kAttentionWorkspaceRows = 65536;

struct AttentionArgs {
  HeadsView q;
  Fp4CacheView cache;
  const int32_t* page_table;
  const int32_t* context_lens;
  const int32_t* q_starts;  // null: one query a sequence
  const int32_t* parents;   // null: each query sees those before it; else a tree of at most 64
  float* workspace;
  uint16_t* out;
  float* lse;  // may be null
  // |scale| * log2(e), at least the smallest normal number (scores of -inf stay that, and finite
  // ones become 0), and the sign bits of a BF16 pair where scale is negative.
  float scale_log2;
  uint32_t q_sign;
  int table_width, seqs, tokens, group, max_q;
  int window;  // 0, or less than the tokens of a page table
};
// Sequences of at most `most` rows, and those of more than `few`.
hipError_t launch_attention_split(const AttentionArgs& args, int dim, int most,
                                  hipStream_t stream);
hipError_t launch_attention_prompt(const AttentionArgs& args, int dim, int few,
                                   hipStream_t stream);
hipError_t launch_attention_tree(const AttentionArgs& args, int dim, hipStream_t stream);
hipError_t launch_attention_fp4(const AttentionArgs& args, int dim, hipStream_t stream);

}  // namespace ci8
