// How attention over the cache is cut into equal runs of tiles, and how the parts of a context are
// joined: shared by the kernels whose waves take tiles of 32 tokens alone (attention_split.hip,
// attention_tree.hip).
#pragma once
#include "attention_device.h"
#include "attention_plan.h"

namespace ci8 {
namespace {

constexpr int kTokens = 32;  // tokens a wave takes at once

// Keeps LDS accesses of a wave's lanes in program order; the LDS itself does.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What the split kernel has of a sequence: blocks of rows, none if those are more than `most`, which
// are the prompt kernel's, and the tiles of each, at least one (it writes the rows that attend to
// nothing). Each block of a key head has its own context.
__device__ __forceinline__ int row_blocks(const Sequence& s, int most, int block_rows) {
  return s.rows > most ? 0 : (s.rows + block_rows - 1) / block_rows;
}
__device__ __forceinline__ int block_tiles(const Sequence& s) { return max(s.tiles(kTokens), 1); }
// What it costs to begin a context, in tiles: queries and pages on their way in and sums out take a
// workgroup 9000 clocks, a tile 800 with three workgroups a CU. Not counted, workgroups that had four
// short contexts ran 73000 clocks where others ran 47000: 32 contexts up to 8000 41 us, counted 37.7,
// 64 from 100 to 4000 58 and 39.
constexpr int kBegin = 10;

// A run: [begin, end) of the row of all sequences' costs, one after the other for each key head and
// block of rows.
struct Run {
  int64_t begin, end, quota;
};
struct Place {
  int seq, head, block, blocks, at, cost;  // at: of its cost
};

// Of 64 sequences from `base` on, one a lane: blocks of a key head, cost of a block, and sums of
// both's products up to each lane's.
struct Counted {
  int base, blocks, cost, sum;
};
__device__ __forceinline__ Counted count_costs(const AttentionArgs& p, int most, int block_rows,
                                               int begin, int lane, int base) {
  Counted c = {base, 0, 1, 0};
  if (base + lane < p.seqs) {
    const Sequence s = sequence(p, base + lane);
    c.blocks = row_blocks(s, most, block_rows);
    c.cost = block_tiles(s) + begin;
  }
  c.sum = wave_scan(c.blocks * c.cost);
  return c;
}
// Costs of all; `first` are those of the first 64 sequences.
__device__ __forceinline__ int64_t all_costs(const AttentionArgs& p, int most, int block_rows,
                                             int begin, int lane, const Counted& first) {
  int64_t total = at_lane(first.sum, 63);
  for (int base = 64; base < p.seqs; base += 64)
    total += at_lane(count_costs(p, most, block_rows, begin, lane, base).sum, 63);
  return total * p.cache.heads;
}

// Where `at` of all costs lies; it is less than their sum. `first`: of the first 64 sequences.
__device__ __forceinline__ Place find_place(const AttentionArgs& p, int most, int block_rows,
                                            int begin, int lane, int64_t at, const Counted& first) {
  const int heads = p.cache.heads;
  Counted c = first;
  int64_t before = 0;
  for (;;) {
    const uint64_t hit = __ballot(before + int64_t(c.sum) * heads > at);
    if (hit || c.base + 64 >= p.seqs) {
      const int which = hit ? __builtin_ctzll(hit) : 0;
      Place place;
      place.seq = uniform(c.base + which);
      place.cost = at_lane(c.cost, which);
      place.blocks = max(at_lane(c.blocks, which), 1);
      const int in_front = at_lane(c.sum, which) - place.cost * place.blocks;
      const int64_t inside = at - before - int64_t(in_front) * heads;
      const int context = uniform(int(inside / place.cost));
      place.at = uniform(int(inside % place.cost));
      place.head = uniform(context / place.blocks);
      place.block = uniform(context % place.blocks);
      return place;
    }
    before += int64_t(at_lane(c.sum, 63)) * heads;
    c = count_costs(p, most, block_rows, begin, lane, c.base + 64);
  }
}

// Parts in the workspace: of workgroup w, part 2w continues a context, part 2w + 1 begins one.
// Sums of rows [part][row][D] first, then their [reference, sum], then what the workgroup that
// begins a context says of it: one for each context (0 parts: its output is written), or, where
// contexts are more than workgroups, for each workgroup, which begins one at most that another
// continues.
struct Joint {
  int parts, first, q_begin, row0, rows, head, unused[2];
};
template <int D, int kTiles>
__device__ __forceinline__ float* part_sums(const AttentionArgs& p, int part) {
  return p.workspace + int64_t(part) * (16 * kTiles * D);
}
template <int D, int kTiles>
__device__ __forceinline__ float* part_stats(const AttentionArgs& p, int part) {
  return p.workspace + int64_t(kAttentionWorkspaceRows) * D + part * (16 * kTiles * 2);
}
template <int D>
__device__ __forceinline__ Joint* joints(const AttentionArgs& p) {
  // the last 64 KiB of the [rows, 2] region
  return reinterpret_cast<Joint*>(p.workspace + int64_t(kAttentionWorkspaceRows) * (D + 2)) - 2048;
}

// The kernel's first argument, read anew: what one part of a long kernel needs of it is not held
// in registers through the others.
__device__ __forceinline__ const AttentionArgs& arguments() {
  auto* args =
      (const __attribute__((address_space(4))) AttentionArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  return *(const AttentionArgs*)args;
}

// Joins the parts of a context (by_context: the blockIdx.x-th, else what workgroup blockIdx.x of the
// split kernel began): 32 channels a workgroup, 8 lanes a row; groups of rows * 8 lanes take every so
// many parts. Bound by the latency of its dependent reads, 1 to 2 us each: the sums of the first
// parts are on their way while the statistics are read, by a row's own lanes where parts are few and
// by whole waves where many.
constexpr int kJoinChannels = 32;
template <int D, int kTiles, int kThreads>
__global__ void __launch_bounds__(kThreads)
    attention_join_kernel(const AttentionArgs p, int most, int most_blocks, int workgroups,
                          bool by_context) {
  constexpr int kRows = 16 * kTiles, kLanes = kJoinChannels / 4, kEarly = 4, kFew = 8;
  static_assert(kRows * kLanes <= kThreads);
  Joint joint = joints<D>(p)[blockIdx.x];
  // Contexts that the split kernel does not have say nothing.
  if (by_context) {
    const int seq = int(blockIdx.x) / most_blocks / p.cache.heads;
    if (int(blockIdx.x) % most_blocks >= row_blocks(sequence(p, seq), most, kRows)) return;
  }
  if (joint.parts <= 0) return;
  // Whatever stands there (a workspace that another stream writes), accesses stay in bounds.
  joint.first = min(max(joint.first, 0), workgroups - 1);
  joint.parts = min(joint.parts, workgroups - joint.first);
  joint.rows = min(max(joint.rows, 1), min(kRows, p.tokens * p.group));
  joint.row0 = min(max(joint.row0, 0), min(most, p.tokens * p.group - joint.rows));
  joint.q_begin = min(max(joint.q_begin, 0),
                      p.tokens - (joint.row0 + joint.rows + p.group - 1) / p.group);
  joint.head = min(max(joint.head, 0), p.cache.heads - 1);
  __shared__ f32x4 sums[kThreads];
  __shared__ float tops[kRows], totals[kRows];
  auto part = [&](int i) { return 2 * (joint.first + i) + (i == 0); };
  const int width = joint.rows * kLanes, groups = kThreads / width;
  const int group = threadIdx.x / width, row = threadIdx.x % width / kLanes;
  const int channel = blockIdx.y * kJoinChannels + threadIdx.x % kLanes * 4;
  auto sum_at = [&](int i) {
    return *reinterpret_cast<const f32x4*>(part_sums<D, kTiles>(p, part(i)) + row * D + channel);
  };
  auto stats_at = [&](int i, int r) {
    return *reinterpret_cast<const f32x2*>(part_stats<D, kTiles>(p, part(i)) + 2 * r);
  };
  f32x4 early[kEarly];
  f32x2 early_stats[kEarly];
#pragma unroll
  for (int e = 0; e < kEarly; ++e) {
    early[e] = f32x4{0, 0, 0, 0};
    early_stats[e] = f32x2{kLowest, 0};
    const int i = group + e * groups;
    if (group < groups && i < joint.parts) {
      early[e] = sum_at(i);
      early_stats[e] = stats_at(i, row);
    }
  }
  float top = kLowest, total = 0;
  if (joint.parts <= kFew) {
    f32x2 stats[kFew];
#pragma unroll
    for (int i = 0; i < kFew; ++i) stats[i] = stats_at(min(i, joint.parts - 1), row);
#pragma unroll
    for (int i = 0; i < kFew; ++i) top = fmaxf(top, stats[i][0]);
#pragma unroll
    for (int i = 0; i < kFew; ++i)
      total += i < joint.parts ? stats[i][1] * __builtin_amdgcn_exp2f(stats[i][0] - top) : 0.f;
  } else {
    const int lane = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < joint.rows; r += kThreads / 64) {
      float m = kLowest, l = 0;
      for (int i = lane; i < joint.parts; i += 64) {
        const f32x2 stats = stats_at(i, r);
        const float most = fmaxf(m, stats[0]);
        l = l * __builtin_amdgcn_exp2f(m - most) +
            stats[1] * __builtin_amdgcn_exp2f(stats[0] - most);
        m = most;
      }
      float most = m;
#pragma unroll
      for (int step = 32; step >= 1; step /= 2) most = fmaxf(most, __shfl_xor(most, step, 64));
      l *= __builtin_amdgcn_exp2f(m - most);
#pragma unroll
      for (int step = 32; step >= 1; step /= 2) l += __shfl_xor(l, step, 64);
      if (lane == 0) {
        tops[r] = most;
        totals[r] = l;
      }
    }
    __syncthreads();
    top = tops[row];
    total = totals[row];
  }
  f32x4 x = {0, 0, 0, 0};
  if (group < groups) {
#pragma unroll
    for (int e = 0; e < kEarly; ++e)
      x += early[e] * __builtin_amdgcn_exp2f(early_stats[e][0] - top);
#pragma unroll 4
    for (int i = group + kEarly * groups; i < joint.parts; i += groups)
      x += sum_at(i) * __builtin_amdgcn_exp2f(stats_at(i, row)[0] - top);
  }
  sums[threadIdx.x] = x;
  __syncthreads();
  if (group == 0) {
    for (int g = 1; g < min(groups, joint.parts); ++g) x += sums[g * width + threadIdx.x];
    write_row4(p, D, joint.q_begin, joint.row0 + row, joint.head, channel, x, top, total);
  }
}

}  // namespace
}  // namespace ci8
