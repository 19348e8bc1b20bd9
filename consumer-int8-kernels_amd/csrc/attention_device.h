// Device helpers shared by the attention kernels (attention_split.hip, attention_prompt.hip).
#pragma once
#include "attention_launch.h"
#include "fp4_device.h"

namespace ci8 {
namespace {

constexpr float kLowest = -3.402823466e38f;
// How far a score may pass the reference, as a power of two of its weight: sums of 2^31 such
// weights stay in FP32, and BF16 weights are as exact at any size.
constexpr float kSlack = 8.f;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Four values of one channel from four token rows, transposed on the way out of LDS: of each 16
// lanes, lanes 4j .. 4j+3 address row j (8 bytes each) and lane i gets column i of the rows.
__device__ __forceinline__ u32x2 lds_read_transposed(const char* p) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (lds_s16x4*)reinterpret_cast<const s16x4*>(p)));
}

// What one sequence asks for.
struct Sequence {
  int q_begin, rows;        // first query row, and rows of (query, head) computed
  int shown;                // queries computed
  int context, shift;       // tokens; position of query 0
  int low, high;            // tokens that any row attends to
  int first_high, last_low; // every row attends to [last_low, first_high)
  __device__ int first_tile(int tokens) const { return low / tokens; }
  __device__ int tiles(int tokens) const {
    return (high + tokens - 1) / tokens - first_tile(tokens);
  }
};

__device__ __forceinline__ Sequence sequence(const AttentionArgs& p, int seq) {
  Sequence s;
  s.q_begin = seq;
  int count = 1;
  if (p.q_starts) {
    s.q_begin = min(max(p.q_starts[seq], 0), p.tokens);
    count = min(max(p.q_starts[seq + 1], s.q_begin), p.tokens) - s.q_begin;
  }
  const int shown = min(count, p.max_q);
  s.shown = shown;
  s.rows = shown * p.group;
  const int64_t capacity = int64_t(p.table_width) << p.cache.page_shift;
  s.context = int(min(int64_t(max(p.context_lens[seq], 0)), capacity));
  s.shift = s.context - count;
  s.high = max(s.shift + shown, 0);
  s.first_high = s.shift + 1;
  s.low = p.window ? max(s.first_high - p.window, 0) : 0;
  s.last_low = p.window ? max(s.high - p.window, 0) : 0;
  return s;
}

// A tree of at most 64 queries. Lane l: the parent of query l as it stands.
__device__ __forceinline__ int tree_parent(const AttentionArgs& p, const Sequence& s, int lane) {
  return lane < s.shown ? p.parents[s.q_begin + lane] : -1;
}
// Lane l gets the set of query l and its ancestors, bit a for query a: sets of parents are joined
// while the way up from each doubles, six rounds at most. A parent is a query before its own; any
// other number is none.
__device__ __forceinline__ uint64_t tree_ancestors(int up, int lane) {
  if (up >= lane) up = -1;
  uint64_t set = lane_set(lane);
  while (__any(up >= 0)) {
    const int from = max(up, 0);
    const uint32_t low = __shfl(int(set), from, 64), high = __shfl(int(set >> 32), from, 64);
    const int next = __shfl(up, from, 64);
    if (up >= 0) {
      set |= uint64_t(high) << 32 | low;
      up = next < 0 ? -1 : next;
    }
  }
  return set;
}

// Those that query l attends to: of its own set a window leaves the last, whose depths are largest.
__device__ __forceinline__ uint64_t tree_seen(const AttentionArgs& p, uint64_t set) {
  if (p.window)
    while (__builtin_popcountll(set) > p.window) set &= set - 1;
  return set;
}
// The first token that query `query` attends to; depths are those of the lanes' queries.
__device__ __forceinline__ int tree_low(const AttentionArgs& p, const Sequence& s, int depth,
                                        int query) {
  return p.window ? max(s.shift + __shfl(depth, query, 64) + 1 - p.window, 0) : 0;
}
// What a row of a tree, which attends to [low, high), sees of the 32 tokens from `first` on, bit i for
// token first + i: those before the tree, and those that its query's set in LDS names. From halves of 32
// bits, as lane_set.
__device__ __forceinline__ uint32_t tree_sees(const uint64_t* seen, int low, int high, int first,
                                              int shift) {
  const uint64_t set = seen[max(high - 1 - shift, 0) & 63];
  const uint32_t near = uint32_t(set), far = uint32_t(set >> 32);
  const int ahead = first - shift;  // the same in all lanes
  uint32_t bits = ~0u;
  if (ahead >= 32)
    bits = ahead < 64 ? far >> (ahead - 32) : 0;
  else if (ahead >= 0)
    bits = __builtin_amdgcn_alignbit(far, near, uint32_t(ahead));
  else if (ahead > -32)
    bits = near << -ahead | ((1u << -ahead) - 1);
  const int passed = low - first;
  if (passed > 0) bits = passed < 32 ? bits >> passed << passed : 0;
  return high > first ? bits : 0;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return int64_t(uint64_t(uint32_t(uniform(int(v)))) | uint64_t(uint32_t(uniform(int(v >> 32)))) << 32);
}

// v of a lane whose number is the same in all.
__device__ __forceinline__ int at_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Inclusive scans of the wave's 64 lanes by DPP (0 beyond the first): rows of 16 by shifts of 1, 2,
// 4 and 8, then the last lane of rows 0 and 2 into rows 1 and 3, of row 1 into rows 2 and 3.
template <int kControl, int kRows>
__device__ __forceinline__ int dpp_or_0(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xF, false);
}
template <typename Op>
__device__ __forceinline__ int wave_scan(int v, Op op) {
  v = op(v, dpp_or_0<0x111, 0xF>(v));
  v = op(v, dpp_or_0<0x112, 0xF>(v));
  v = op(v, dpp_or_0<0x114, 0xF>(v));
  v = op(v, dpp_or_0<0x118, 0xF>(v));
  v = op(v, dpp_or_0<0x142, 0xA>(v));
  return op(v, dpp_or_0<0x143, 0xC>(v));
}
__device__ __forceinline__ int wave_scan(int v) {
  return wave_scan(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_sum(int v) { return at_lane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_max(int v) {  // of values that are not negative
  return at_lane(wave_scan(v, [](int a, int b) { return max(a, b); }), 63);
}

__device__ __forceinline__ void write_row4(const AttentionArgs& p, int dim, int q_begin, int row,
                                           int kv_head, int channel, const f32x4& x, float top,
                                           float sum) {
  const float inv = sum == 0 ? 0.f : 1.f / sum;
  const int64_t at = int64_t(q_begin + row / p.group) * p.q.heads + kv_head * p.group +
                     row % p.group;
  *reinterpret_cast<u32x2*>(p.out + at * dim + channel) =
      u32x2{pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv)};
  if (p.lse && channel == 0)
    p.lse[at] =
        sum == 0 ? -__builtin_inff() : (top + __builtin_log2f(sum)) * 0.693147180559945309f;
}

}  // namespace
}  // namespace ci8
