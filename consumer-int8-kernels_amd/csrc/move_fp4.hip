// move_fp4 (include/consumer_int8_drafts.h): cache rows of a sequence to earlier rows of it, as they
// are, keys and values of all heads.
//
// A row of a head is 16-byte pieces of codes, and its scales: a thread has one piece of one head for
// all rows of a sequence, in order, so that what a later row reads is never written before. Rows to
// move are few (the accepted ones of a tree), so this is bound by its chain of loads: a row's
// number, its slot, its bytes. 64 rows are looked up at once, one a lane, and four copied at a time: 32
// sequences of 26 rows in a tree, 8 heads of 128, 3.6 us, most of it the launch and these loads.
#include "attention_launch.h"
#include "attention_plan.h"
#include "fp4_device.h"

namespace ci8 {
namespace {

__device__ __forceinline__ int at_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

template <int D>
__global__ void __launch_bounds__(kMoveThreads)
    move_fp4_kernel(const Fp4CacheView cache, const int32_t* __restrict__ rows,
                    const int64_t* __restrict__ slots, const int32_t* __restrict__ q_starts,
                    int tokens, int blocks) {
  constexpr int kPieces = D / kFp4Block, kScales = D / kFp4Block;  // 16 bytes each; bytes of a row
  const int seq = blockIdx.x / blocks, lane = threadIdx.x & 63;
  const int begin = min(max(q_starts[seq], 0), tokens);
  const int count = min(max(q_starts[seq + 1], begin), tokens) - begin;

  // The thread's part of a row; threads past the last have none.
  const int index = blockIdx.x % blocks * kMoveThreads + threadIdx.x;
  const int head = index / (2 * (kPieces + 1)), part = index % (2 * (kPieces + 1));
  const bool live = head < cache.heads;
  const Fp4Rows& side = part > kPieces ? cache.v : cache.k;
  const int piece = part % (kPieces + 1);
  const bool scales = piece == kPieces;
  uint8_t* const base = (scales ? side.scales : side.codes + 16 * piece) +
                        (int64_t(live ? head : 0) << cache.page_shift) * (scales ? kScales : D / 2);
  const int64_t stride = scales ? side.scale_stride : side.code_stride;
  const int pitch = scales ? kScales : D / 2;

  for (int first = 0; first < count; first += 64) {
    // Lane l: row first + l, where it comes from and goes to.
    int from_page = 0, from_row = 0, to_page = 0, to_row = 0;
    bool moves = false;
    if (first + lane < count) {
      const int source = rows[begin + first + lane];
      if (source > first + lane && source < count) {
        const int64_t from = slots[begin + source], to = slots[begin + first + lane];
        const int64_t all = int64_t(cache.pages) << cache.page_shift;
        moves = from >= 0 && from < all && to >= 0 && to < all;
        const int mask = (1 << cache.page_shift) - 1;
        from_page = int(from >> cache.page_shift);
        from_row = int(from) & mask;
        to_page = int(to >> cache.page_shift);
        to_row = int(to) & mask;
      }
    }
    uint64_t left = __ballot(moves);
    while (left) {
      constexpr int kAtOnce = 4;
      u32x4 data[kAtOnce];
      uint8_t* to[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        to[i] = nullptr;
        if (!left) continue;
        const int l = __builtin_ctzll(left);
        left &= left - 1;
        const uint8_t* from = base + at_lane(from_page, l) * stride + at_lane(from_row, l) * pitch;
        to[i] = base + at_lane(to_page, l) * stride + at_lane(to_row, l) * pitch;
        if (!live) continue;
        if (!scales)
          data[i] = *reinterpret_cast<const u32x4*>(from);
        else if constexpr (D == 64)
          data[i][0] = *reinterpret_cast<const uint16_t*>(from);
        else if constexpr (D == 128)
          data[i][0] = *reinterpret_cast<const uint32_t*>(from);
        else
          *reinterpret_cast<u32x2*>(&data[i]) = *reinterpret_cast<const u32x2*>(from);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (!live || !to[i]) continue;
        if (!scales)
          *reinterpret_cast<u32x4*>(to[i]) = data[i];
        else if constexpr (D == 64)
          *reinterpret_cast<uint16_t*>(to[i]) = uint16_t(data[i][0]);
        else if constexpr (D == 128)
          *reinterpret_cast<uint32_t*>(to[i]) = data[i][0];
        else
          *reinterpret_cast<u32x2*>(to[i]) = *reinterpret_cast<const u32x2*>(&data[i]);
      }
    }
  }
}

}  // namespace

hipError_t launch_move_fp4(const Fp4CacheView& cache, const int32_t* rows, const int64_t* slots,
                           const int32_t* q_starts, int seqs, int tokens, int dim,
                           hipStream_t stream) {
  if (seqs == 0 || tokens == 0) return hipSuccess;
  const int blocks = int(move_blocks(cache.heads, dim));
  const auto kernel = dim == 64    ? move_fp4_kernel<64>
                      : dim == 128 ? move_fp4_kernel<128>
                                   : move_fp4_kernel<256>;
  kernel<<<uint32_t(seqs) * blocks, kMoveThreads, 0, stream>>>(cache, rows, slots, q_starts, tokens,
                                                              blocks);
  return hipGetLastError();
}

}  // namespace ci8
