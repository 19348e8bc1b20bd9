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
  // with one: 4096 tokens of 24 + 4 heads of 256 28.2 and 31.8, 9261 of 16 + 16 of 64 with three
  // axes 23.4 and 51.2; but 1024 of 32 + 8 of 128 8.6 and 8.3, 64 of them 5.3 and 3.0.
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

}  // namespace ci8
