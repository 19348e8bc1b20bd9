// Sizes of the attention operators' launches, shared by the checks of attention_abi.cpp and the
// launchers. Plain C++, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

namespace ci8 {

// HIP takes fewer than 2^32 work-items along x.
constexpr bool launch_fits(int64_t workgroups, int threads) {
  return workgroups <= ((int64_t(1) << 32) - 1) / threads;
}

// qk_norm_rope and append_fp4: a group is the 512 / dim heads of queries, of keys or of values that a
// wave takes at once, a chunk the groups of one token that a wave has, four waves a workgroup.
constexpr int kNormThreads = 256;
struct NormRopeGrid {
  int q_groups, k_groups, groups, per_wave, chunks;
  int64_t workgroups;
};
inline NormRopeGrid norm_rope_grid(int64_t tokens, int q_heads, int k_heads, int dim, bool append) {
  const int heads = 512 / dim;
  NormRopeGrid g = {};
  g.q_groups = (q_heads + heads - 1) / heads;
  g.k_groups = (k_heads + heads - 1) / heads;
  g.groups = g.q_groups + g.k_groups * (append ? 2 : 1);
  // Four groups a wave, which share its angles, once waves are many. Microseconds with four and
  // with one, in a graph: 9261 tokens of 16 + 16 heads of 64 with three axes 20.3 and 35.2; with one axis
  // little between them, 4096 of 24 + 4 of 256 24.1 and 23.9, of 32 + 8 of 128 20.4 and 18.7; but 300 of
  // 40 + 8 of 128 5.7 and 4.1, 64 of 32 + 8 5.2 and 3.1.
  g.per_wave = tokens * g.groups >= 32768 ? 4 : 1;
  g.chunks = (g.groups + g.per_wave - 1) / g.per_wave;
  g.workgroups = (tokens * g.chunks + 3) / 4;
  return g;
}

// unpack_fp4: a thread for 8 channels.
constexpr int kUnpackThreads = 256;
inline int64_t unpack_workgroups(int64_t count, int heads, int dim) {
  return (count * heads * (dim / 8) + kUnpackThreads - 1) / kUnpackThreads;
}

// attention_fp4: rows are (token, query head of one key head) pairs. Sequences of at most `few` rows go
// to the split kernel, the others to the prompt kernel.
//
// Up to kMostRows they are few: above 32 in blocks that each read the cache, which the caches between
// them and HBM mostly hold. With the prompt kernel's 256 rows a workgroup instead, us: 16 x 5 tokens
// behind contexts up to 16000 of 64 query and 8 key heads of 128 79 and 214, 16 tokens each 145 and
// 220; 16 x 100 rows of 16 heads of 64 199 and 268, 48 rows 109 and 267. Above, blocks and the prompt
// kernel: 4 x 32 tokens (256 rows) behind up to 30000 133 and 122, 16 x 32 277 and 235, 2 x 200 rows at 64
// channels 61 and 49; but 8 x 150 132 and 145, 4 x 32 tokens (192 rows) of 24 and 4 heads of 256 65 and 85.
constexpr int kMostRows = 128;
struct RowSplit {
  int few;
  bool split, prompt;  // which kernels may have sequences
};
inline RowSplit row_split(int64_t tokens, int64_t seqs, int group, int64_t max_q) {
  // Beside prompts `few` is 16 or 32, so that the usual decode fits.
  const int64_t most = max_q * group;
  int few = most <= kMostRows ? int(most) : group <= 16 ? 16 : 32;
  // No sequence can be that short where all others at their longest leave more than that: then
  // the prompt kernel has them all.
  if (most > few && (tokens - (seqs - 1) * max_q) * group > few) few = 0;
  return {few, group <= few, most > few};
}

// Units of the prompt kernel's work at most: its row tiles (each but a sequence's last is full) for
// each key head. The kernel has as many workgroups, and one more a CU where contexts may be cut.
constexpr int kPromptRows = 256, kPromptThreads = 512;
inline int64_t prompt_units(int64_t tokens, int64_t seqs, int group, int64_t max_q, int heads) {
  const int64_t each = (max_q * group + kPromptRows - 1) / kPromptRows;
  const int64_t bound = tokens * group / kPromptRows + seqs;
  return (bound < each * seqs ? bound : each * seqs) * heads;
}

}  // namespace ci8
