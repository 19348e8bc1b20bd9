// attention_fp4 for many query rows a sequence (include/consumer_int8_attention.h): prompts, and
// chunks of them behind a context.
//
// The mathematics and the order of operands are attention_split.hip's, with 32 x 32 x 16 MFMAs:
// S^T = K Q^T leaves a row's scores in the registers of its column's two lanes, where they are
// weighted and become the operand of O^T += V^T P^T without an exchange. Rows are (token, query
// head of one key head) pairs, 256 a workgroup, so that heads that share a key head share its
// tiles. Four operations a score and channel: bound by the MFMA rate, then by the softmax's
// vector instructions (by the counters 7.8 for each MFMA at 128 channels, which is each register of
// scores; masks, staging and addresses counted) and by LDS reads (each wave reads every tile). Two waves a
// SIMD of 32 rows each, in alternate phases: the scores of the next tile are on the matrix unit while
// the vector unit weighs those of this one. Measured: 4096 tokens of 40 query and 8 key heads of 128
// 192 us (199 on another card), 895 TFLOP/s of what the mask leaves (a large product reaches 1157 to
// 1265); 24 and 4 of 256 242 us, 853 (415 us with one wave a SIMD that holds all its queries); 16 heads of
// 64 81 us, 423, and 14 and 2 of 64 behind 8000 more 209 us, 687: half the MFMAs for as many scores.
// Weights are rounded to BF16 for the second product as in attention_split.hip.
//
// Tiles of keys and values are converted to BF16 once a workgroup, on their way into LDS: global
// loads run two tiles ahead, one barrier a tile.
#include <type_traits>

#include "attention_device.h"
#include "attention_plan.h"
#include "launch.h"
#include "prompt_schedule.h"

namespace ci8 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Rows of a workgroup in tiles of 32, its waves, and tokens of a tile.
template <int D>
struct Shape {
  static constexpr int kTiles = 1;  // of a wave
  static constexpr int kWaves = 8;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRows = 32 * kTiles * kWaves;
  static_assert(kRows == kPromptRows && kThreads == kPromptThreads);
  static constexpr int kTokens = D == 64 ? 128 : D == 128 ? 64 : 32;
  static constexpr int kBlocks = D / kFp4Block;
  // Byte pitch of LDS rows of keys: 16 of them, 16 bytes each, fall on different banks. Rows of
  // values are not padded; their pieces trade places instead (value_at), so that transposed
  // reads of 64 bytes of 4 tokens, and writes of 16 lanes' pieces, fall on different banks.
  static constexpr int kKeyPitch = 2 * D + 16, kValuePitch = 2 * D;
  static constexpr int kKeyBytes = kTokens * kKeyPitch, kValueBytes = kTokens * kValuePitch;
  static constexpr int kPacks = 2 * kTokens * kBlocks / kThreads;  // 16 bytes of codes a thread
  static_assert(2 * kTokens * kBlocks % kThreads == 0);
  static constexpr int kHalves = kTokens / 32;
  static_assert(schedule_holds(kHalves, barrier_half(kHalves)), "LDS buffers are not raced for");
  static constexpr int kLdsBytes = kKeyBuffers * kKeyBytes + kValueBuffers * kValueBytes;
  static_assert(kKeyBuffers * kKeyBytes % 256 == 0);
  // Byte of piece j (8 channels) of a token's block in a buffer of values: among the 256 bytes
  // that hold it, blocks are XORed by the token, and in a block the pieces are.
  __device__ static constexpr int value_at(int token, int block, int j) {
    return D == 64 ? token * kValuePitch + 64 * (block ^ (token >> 1 & 1)) +
                         16 * (j ^ (token >> 1 & 3))
                   : token * kValuePitch + 256 * (block / 4) + 64 * (block % 4 ^ token % 4) +
                         16 * (j ^ (D == 128 ? token % 4 : token % 2 * 2 + block / 4));
  }
};

// Row tiles of a sequence that this kernel has.
__device__ __forceinline__ int row_tiles(const Sequence& s, int few, int rows) {
  return s.rows <= few ? 0 : (s.rows + rows - 1) / rows;
}

// Row tiles of all sequences, and the one that `index` counts to.
struct RowTile {
  int seq, tile, tiles;  // seq < 0: past the last
};
__device__ __forceinline__ int all_row_tiles(const AttentionArgs& p, int few, int rows, int lane) {
  int total = 0;
  for (int base = 0; base < p.seqs; base += 64) {
    int n = 0;
    if (base + lane < p.seqs) n = row_tiles(sequence(p, base + lane), few, rows);
    total += wave_sum(n);
  }
  return total;
}
__device__ __forceinline__ RowTile find_row_tile(const AttentionArgs& p, int few, int rows,
                                                 int index, int lane) {
  for (int base = 0; base < p.seqs; base += 64) {
    int n = 0;
    if (base + lane < p.seqs) n = row_tiles(sequence(p, base + lane), few, rows);
    const int sum = wave_scan(n);
    const uint64_t hit = __ballot(sum > index);
    if (hit) {
      const int which = __builtin_ctzll(hit);
      const int tiles = at_lane(n, which);
      return {base + which, index - (at_lane(sum, which) - tiles), tiles};
    }
    index -= at_lane(sum, 63);
  }
  return {-1, 0, 0};
}

// Units of work are (row tile, key head). One a CU, they run in rounds; those of a last round that
// does not fill the GPU have their contexts cut, so that it does.
struct Cut {
  int units, whole, splits;  // units from `whole` on are cut
};
__device__ __forceinline__ Cut cut_units(const AttentionArgs& p, int few, int rows, int cus,
                                         int most_splits, int lane) {
  Cut c;
  c.units = all_row_tiles(p, few, rows, lane) * p.cache.heads;
  const int rest = c.units % cus;
  c.whole = c.units - rest;
  c.splits = rest ? min(cus / rest, most_splits) : 1;
  if (c.splits <= 1) {
    c.splits = 1;
    c.whole = c.units;
  }
  return c;
}

// Parts of the workspace: [cut unit][split][row][D] and the statistics after them.
__device__ __forceinline__ float* part_sums(const AttentionArgs& p, int64_t row, int dim) {
  return p.workspace + row * dim;
}
__device__ __forceinline__ float* part_stats(const AttentionArgs& p, int64_t row, int dim) {
  return p.workspace + int64_t(kAttentionWorkspaceRows) * dim + row * 2;
}

template <int D>
__global__ void __launch_bounds__(Shape<D>::kThreads)
    attention_prompt_kernel(const AttentionArgs p, int few, int cus, int most_splits) {
  using S = Shape<D>;
  constexpr int kTokens = S::kTokens, kTiles = S::kTiles, kHalves = S::kHalves;
  constexpr int kSteps = D / 16, kChannels = D / 32;
  // The waves' queries stay in registers; where the sums leave room for half of them, the others are
  // in LDS.
  constexpr int kHeld = D == 256 ? kSteps / 2 : kSteps;
  __shared__ u32x4 late_q[D == 256 ? (kSteps - kHeld) * S::kThreads : 1];
  // The buffers of keys, then those of values.
  __shared__ __align__(256) char lds[S::kLdsBytes];
  constexpr int kValues = kKeyBuffers * S::kKeyBytes;
  __shared__ uint8_t poison[kPoisonBuffers][kTokens][S::kBlocks];  // NaN blocks of edge tiles
  __shared__ int poisoned[kPoisonBuffers];  // the last such tile that has any

  const int thread = threadIdx.x, lane = thread & 63, wave = uniform(thread >> 6);
  const int column = lane & 31, half = lane >> 5;
  const int heads = p.cache.heads;
  int unit = blockIdx.x, split = 0, splits = 1, part = 0;
  if (most_splits > 1) {
    const Cut c = cut_units(p, few, S::kRows, cus, most_splits, lane);
    if (unit >= c.whole) {
      splits = c.splits;
      part = unit - c.whole;
      unit = c.whole + part / splits;
      split = part % splits;
    }
  }
  const int kv_head = unit % heads;
  const RowTile where = find_row_tile(p, few, S::kRows, unit / heads, lane);
  if (where.seq < 0) return;
  const Sequence s = sequence(p, where.seq);
  // The last rows see the most: they go first.
  const int row0 = (where.tiles - 1 - where.tile) * S::kRows;
  const int last_row = min(row0 + S::kRows, s.rows) - 1;

  // Tokens that any row of the workgroup attends to, and those that all attend to.
  const int first_high = s.shift + row0 / p.group + 1, high = max(s.shift + last_row / p.group + 1, 0);
  const int tile_low = p.window ? max(first_high - p.window, 0) : 0;
  const int last_low = p.window ? max(high - p.window, 0) : 0;
  int t_begin = tile_low / kTokens, t_end = (high + kTokens - 1) / kTokens;
  if (splits > 1) {
    const int n = max(t_end - t_begin, 0), each = (n + splits - 1) / splits;
    const int end = t_end;
    t_begin = min(t_begin + split * each, end);
    t_end = min(t_begin + each, end);
  }

  const int context_page = max(s.context - 1, 0) >> p.cache.page_shift;
  const int32_t* const table = p.page_table + int64_t(where.seq) * p.table_width;
  // Staging. A thread converts 32 channels of one token a pack; a wave's packs are all of the keys
  // or all of the values, of one page or two. Pages are looked up a tile ahead of the codes, these
  // are loaded a tile ahead of their use. Past the last tile this goes on with tokens that are
  // there, into buffers that nobody reads, since branches would cost more.
  constexpr int kPerTile = kTokens * S::kBlocks, kWaveTokens = 64 / S::kBlocks;
  constexpr bool kTwoPages = kWaveTokens > 16;
  static_assert(kPerTile % 64 == 0 && kWaveTokens <= 32);
  struct Staged {
    u32x4 codes[S::kPacks];
    uint32_t scales[S::kPacks];
  };
  struct Pages {
    int at[S::kPacks];
  };
  const int lane_token = lane / S::kBlocks, block = lane % S::kBlocks;
  const int page_mask = (1 << p.cache.page_shift) - 1;
  // Scales are loaded as the words that hold them: a loop-carried byte would be masked, and so
  // waited for, at the loop's end.
  const uint32_t scale_byte = lane_token % 16 * S::kBlocks + block;
  const uint32_t scale_turn = fp4_scale_turn(scale_byte % 4);
  // The lane's bytes from its row of 16 tokens on.
  const uint32_t code_at = lane_token % 16 * (D / 2) + 16 * block, scale_at = scale_byte & ~3u;
  struct Pack {
    bool value;
    int token;                // the wave's first in a tile
    const uint8_t *codes, *scales;  // of this head's rows in page 0
    int64_t code_stride, scale_stride;
    int to;                   // LDS byte of the lane's first piece in the first buffer
  };
  auto pack = [&](int c) __attribute__((always_inline)) {
    Pack x;
    x.value = c * S::kThreads + 64 * wave >= kPerTile;
    x.token = (c * S::kThreads + 64 * wave) % kPerTile / S::kBlocks;
    const Fp4Rows& rows = x.value ? p.cache.v : p.cache.k;
    const int64_t row = int64_t(kv_head) << p.cache.page_shift;
    x.codes = rows.codes + row * (D / 2);
    x.scales = rows.scales + row * S::kBlocks;
    x.code_stride = rows.code_stride;
    x.scale_stride = rows.scale_stride;
    const int token = x.token + lane_token;
    x.to = x.value ? kValues + S::value_at(token, block, 0) : token * S::kKeyPitch + 64 * block;
    return x;
  };
  Pack packs[S::kPacks];
#pragma unroll
  for (int c = 0; c < S::kPacks; ++c) packs[c] = pack(c);
  // Makes page lookups vector loads: scalar ones would be waited for with every LDS read.
  int lane_zero = 0;
  asm volatile("" : "+v"(lane_zero));
  // Tiles of the keys and of the values.
  auto load_pages = [&](Pages& pages, int tk, int tv) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) {
      const int token = (packs[c].value ? tv : tk) * kTokens + packs[c].token;
      const int at = (kTwoPages ? token + (lane_token & 16) : token + lane_zero) >> p.cache.page_shift;
      pages.at[c] = table[min(at, context_page)];
    }
  };
  auto load_codes = [&](Staged& staged, const Pages& pages, int tk, int tv)
      __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) {
      const Pack& x = packs[c];
      const int token = (x.value ? tv : tk) * kTokens + x.token;
      auto offsets = [&](int page, int first, int64_t& code, int64_t& scale)
          __attribute__((always_inline)) {
        // Loads stay in the cache.
        const int64_t at = uint32_t(page) < uint32_t(p.cache.pages) ? page : 0;
        const int row = first & page_mask;
        code = at * x.code_stride + row * (D / 2);
        scale = at * x.scale_stride + row * S::kBlocks;
      };
      int64_t code, scale;
      offsets(uniform(pages.at[c]), token, code, scale);
      if constexpr (kTwoPages) {
        int64_t code2, scale2;
        offsets(at_lane(pages.at[c], 16 * S::kBlocks), token + 16, code2, scale2);
        code = lane_token >= 16 ? code2 : code;
        scale = lane_token >= 16 ? scale2 : scale;
      }
      staged.codes[c] = *reinterpret_cast<const u32x4*>(x.codes + code + code_at);
      staged.scales[c] = *reinterpret_cast<const uint32_t*>(x.scales + scale + scale_at);
    }
  };

  // The way in: pages, queries and codes are all on their way before the first wait for HBM but one.
  Staged staged, ahead;
  Pages pages, pages_ahead, pages_first;
  if (t_begin < t_end) {
    load_pages(pages_first, t_begin, t_begin);
    load_pages(pages_ahead, t_begin + 1, t_begin);
    load_pages(pages, t_begin + 2, t_begin + 1);
  }
  // Pages outside the cache are rare: whether there are any is found once.
  bool missing = false;
  if (t_begin < t_end) {
    const int last = min((t_end * kTokens - 1) >> p.cache.page_shift, context_page);
    for (int i = (t_begin * kTokens >> p.cache.page_shift) + thread; i <= last; i += S::kThreads)
      missing = missing || uint32_t(table[i]) >= uint32_t(p.cache.pages);
  }
  // The lane's rows and their tokens [low, high). Lanes past the last row repeat it; their results
  // go nowhere.
  int row_low[kTiles], row_high[kTiles];
  u32x4 q[kTiles][kHeld];
  const int wave_row = row0 + wave * 32 * kTiles;
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int row = min(wave_row + 32 * n + column, s.rows - 1), query = row / p.group;
    row_high[n] = s.shift + query + 1;
    row_low[n] = p.window ? max(row_high[n] - p.window, 0) : 0;
    const uint16_t* src = p.q.data + int64_t(s.q_begin + query) * p.q.token_stride +
                          int64_t(kv_head * p.group + row % p.group) * p.q.head_stride;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(src + 16 * j + 8 * half) ^ p.q_sign;
      if (j < kHeld)
        q[n][j] = x;
      else
        late_q[(j - kHeld) * S::kThreads + thread] = x;
    }
  }
  if (t_begin < t_end) {
    load_codes(staged, pages_first, t_begin, t_begin);
    load_codes(ahead, pages_ahead, t_begin + 1, t_begin);
  }
  // Tokens [all_low, all_high) that all of the wave's rows attend to.
  const int all_high = s.shift + min(wave_row, s.rows - 1) / p.group + 1;
  const int any_high = s.shift + min(wave_row + 32 * kTiles - 1, s.rows - 1) / p.group + 1;
  const int all_low = p.window ? max(any_high - p.window, 0) : 0;

  f32x16 o[kTiles][kChannels];
  float reference[kTiles], limit[kTiles], sum[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
#pragma unroll
    for (int m = 0; m < kChannels; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][m][i] = 0;
    reference[n] = 0;
    limit[n] = kLowest;
    sum[n] = 0;
  }

  if (thread < kPoisonBuffers) poisoned[thread] = -1;
  const bool any_missing = __syncthreads_or(missing);

  auto there = [&](int token) __attribute__((always_inline)) {
    return uint32_t(table[min(token >> p.cache.page_shift, context_page)]) < uint32_t(p.cache.pages);
  };
  auto edge_tile = [&](int t) __attribute__((always_inline)) {
    return (t + 1) * kTokens > first_high || t * kTokens < last_low;
  };
  // key_buffer: where tile tk goes, one of the three in turn.
  auto store_tiles = [&](const Staged& staged, int key_buffer, int tv) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) {
      const Pack& x = packs[c];
      u32x4 codes = staged.codes[c];
      uint32_t scales = staged.scales[c];
      if (x.value && (edge_tile(tv) || any_missing)) {
        // Values of no page or past the context are zeros, and so are an edge tile's NaN blocks.
        const int token = tv * kTokens + x.token + lane_token;
        const bool real = token < s.context && (!any_missing || there(token));
        const bool nan = real && (scales >> scale_byte % 4 * 8 & 0xFF) >= 253 && edge_tile(tv);
        poison[tv % kPoisonBuffers][x.token + lane_token][block] = nan;
        if (nan) poisoned[tv % kPoisonBuffers] = tv;
        codes = nan || !real ? u32x4{0, 0, 0, 0} : codes;
        scales = nan || !real ? 0 : scales;
      }
      const int buffer = x.value ? int(uint32_t(tv) % kValueBuffers) * S::kValueBytes : key_buffer * S::kKeyBytes;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<u32x4*>(
            lds + (((x.to + buffer) ^ (x.value ? 16 * j : 0)) + (x.value ? 0 : 16 * j))) =
            fp4_to_bf16x8(codes[j], fp4_scale_in(scales, scale_turn));
    }
  };

  // Half b of tile t is 32 tokens. Where registers allow, operands are read from LDS half a step
  // before their products.
  constexpr bool kAhead = kHalves > 1;
  constexpr int kKeysAhead = keys_ahead(kHalves), kValuesAhead = values_ahead(kHalves);
  u32x4 key[kSteps];
  auto read_keys = [&](int buffer, int b) __attribute__((always_inline)) {
    const char* from = lds + buffer * S::kKeyBytes + (32 * b + column) * S::kKeyPitch + 16 * half;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) key[j] = *reinterpret_cast<const u32x4*>(from + 32 * j);
  };
  auto multiply = [&](f32x16(&score)[kTiles]) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) score[n][i] = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
        score[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, key[j]), __builtin_bit_cast(bf16x8, q[n][j]), score[n], 0,
            0, 0);
  };

  // Scores become exponents x = s * scale - reference; most: the lane's largest.
  float most[kTiles];
  auto largest = [&](const f32x16& x) __attribute__((always_inline)) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) m = fmaxf(m, x[i]);
    return m;
  };
  auto scale = [&](f32x16(&score)[kTiles]) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) score[n][i] = fmaf(score[n][i], p.scale_log2, -reference[n]);
      most[n] = largest(score[n]);
    }
  };
  // Hides what rows do not attend to, and moves their references where exponents pass the limit:
  // kSlack, and anything for a row that has seen nothing.
  auto settle = [&](int first, f32x16(&x)[kTiles]) __attribute__((always_inline)) {
    const bool edge = first > all_high - 32 || first < all_low || any_missing;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      if (edge) {
        const bool low_there = !any_missing || there(first);
        const bool high_there = !any_missing || there(first + 16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 8 * (i / 4) + i % 4, token = first + at + 4 * half;
          const bool seen = (token >= row_low[n]) & (token < row_high[n]) &
                            (at < 16 ? low_there : high_there);
          x[n][i] = seen ? x[n][i] : -__builtin_inff();
        }
        most[n] = largest(x[n]);
      }
      if (__any(most[n] > limit[n])) {
        const float m = fmaxf(most[n], __shfl_xor(most[n], 32, 64));
        const bool fresh = limit[n] < 0;
        float next = reference[n];
        if (fresh ? m > kLowest : m > 0) next += m;
        const float up = next - reference[n];
        const float factor = fresh ? 1.f : __builtin_amdgcn_exp2f(-up);
        if (m > kLowest) limit[n] = kSlack;
        reference[n] = next;
        sum[n] *= factor;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[n][i] -= up;
#pragma unroll
        for (int c = 0; c < kChannels; ++c) o[n][c] *= factor;
      }
    }
  };
  u32x4 weights[kTiles][2];
  auto weigh = [&](f32x16(&x)[kTiles]) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float total[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[n][i] = __builtin_amdgcn_exp2f(x[n][i]);
        total[i % 2] += x[n][i];
      }
      sum[n] += total[0] + total[1];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          weights[n][c][i] = pack_bf16x2(x[n][8 * c + 2 * i], x[n][8 * c + 2 * i + 1]);
    }
  };
  u32x4 value[2][kChannels];
  auto read_value = [&](int t, int b, int c, int m) __attribute__((always_inline)) {
    // The lane's row of four and its 8 bytes of the 64 that two groups of 16 lanes read: piece
    // 2 * (lane / 16 % 2) + lane % 4 / 2. Tokens of other fours keep its place in the row.
    const int row = 4 * half + lane % 16 / 4, piece = 2 * (lane / 16 % 2) + lane % 4 / 2;
    const char* at = lds + (kValues + int(uint32_t(t) % kValueBuffers) * S::kValueBytes + 32 * b * S::kValuePitch) +
                     lane % 2 * 8 + S::value_at(row, m, piece) + 16 * c * S::kValuePitch;
    const u32x2 x = lds_read_transposed(at);
    const u32x2 y = lds_read_transposed(at + 8 * S::kValuePitch);
    return u32x4{x[0], x[1], y[0], y[1]};
  };
  auto read_values = [&](int t, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < kChannels; ++m) value[c][m] = read_value(t, b, c, m);
  };
  auto add_values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          o[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, value[c][m]), __builtin_bit_cast(bf16x8, weights[n][c]),
              o[n][m], 0, 0, 0);
  };
  // NaN blocks of an edge tile's values stand as zeros; rows that see their token get the NaN.
  auto add_poison = [&](int t) __attribute__((always_inline)) {
    for (int token = 0; token < kTokens; ++token)
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
        if (poison[t % kPoisonBuffers][token][m]) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
            if (t * kTokens + token >= row_low[n] && t * kTokens + token < row_high[n])
              o[n][m] += __builtin_nanf("");
        }
  };

  f32x16 scores[kTiles];
  static_assert(kAhead ? kHeld == kSteps : kTiles == 1);
  // At D = 256 operands are read where they are used, a few at a time: all of a tile's would not fit
  // beside the sums.
  auto stream_scores = [&](int buffer) __attribute__((always_inline)) {
    const char* from = lds + buffer * S::kKeyBytes + column * S::kKeyPitch + 16 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) scores[0][i] = 0;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const u32x4 query = j < kHeld ? q[0][j] : late_q[(j - kHeld) * S::kThreads + thread];
      scores[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(from + 32 * j)),
          __builtin_bit_cast(bf16x8, query), scores[0], 0, 0, 0);
      if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto stream_values = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < kChannels; ++m) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
        o[0][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, read_value(t, 0, c, m)),
            __builtin_bit_cast(bf16x8, weights[0][c]), o[0][m], 0, 0, 0);
      if (m % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (t_begin < t_end) {
    // In a tile's step the keys of the next tile but one are staged, and the values of the next.
    static_assert(kKeysStaged == 2 && kValuesStaged == 1);
    store_tiles(staged, 0, t_begin);
    load_codes(staged, pages, t_begin + 2, t_begin + 1);
    load_pages(pages, t_begin + 3, t_begin + 2);
    store_tiles(ahead, 1, t_begin);
    __syncthreads();
    if (kAhead) {
      read_keys(0, 0);
      multiply(scores);
    } else {
      stream_scores(0);
    }
    scale(scores);
    if (kAhead) {
      read_keys(1 / kHalves, 1 % kHalves);
      read_values(t_begin, 0);
    }
  }
  int buffer[3] = {0, 1, 2};  // of the keys of this tile and the next two
  for (int t = t_begin; t < t_end; ++t) {
#pragma unroll
    for (int b = 0; b < kHalves; ++b) {
      // Weighs this half's scores, and stages what the next halves read.
      settle(t * kTokens + 32 * b, scores);
      weigh(scores);
      if (b == 0) store_tiles(staged, buffer[2], t + 1);
      // This half's values, the next half's scores (past the last tile those of old keys, which
      // nothing reads), and the operands after those.
      __builtin_amdgcn_s_setprio(1);
      if (kAhead)
        multiply(scores);
      else
        stream_scores(buffer[1]);
      if (kAhead) read_keys(buffer[(b + kKeysAhead) / kHalves], (b + kKeysAhead) % kHalves);
      if (kAhead)
        add_values();
      else
        stream_values(t);
      if (kAhead) read_values(t + (b + kValuesAhead) / kHalves, (b + kValuesAhead) % kHalves);
      scale(scores);
      if (b == 0) {
        load_codes(staged, pages, t + 3, t + 2);
        load_pages(pages, t + 4, t + 3);
      }
      // LDS reads and vector instructions go between the MFMAs.
      if (kAhead) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < 2 * kChannels; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (b + 1 == kHalves && edge_tile(t) && poisoned[t % kPoisonBuffers] == t) add_poison(t);
      // One barrier a tile, where it parts what is stored from what is read (prompt_schedule.h): with
      // one or two halves at the end of the first, with four of the third.
      if (b == barrier_half(kHalves)) {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int first = buffer[0];
    buffer[0] = buffer[1];
    buffer[1] = buffer[2];
    buffer[2] = first;
  }

  // A row's two lanes hold the sums of their own tokens.
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const float total = sum[n] + __shfl_xor(sum[n], 32, 64);
    const float top = limit[n] < 0 ? kLowest : reference[n];
    const int row = wave_row + 32 * n + column;
    if (row >= s.rows) continue;
    if (splits == 1) {
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = {o[n][m][4 * i], o[n][m][4 * i + 1], o[n][m][4 * i + 2], o[n][m][4 * i + 3]};
          write_row4(p, D, s.q_begin, row, kv_head, 32 * m + 8 * i + 4 * half, x, top, total);
        }
    } else {
      const int64_t at = int64_t(part) * S::kRows + (row - row0);
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(part_sums(p, at, D) + 32 * m + 8 * i + 4 * half) =
              f32x4{o[n][m][4 * i], o[n][m][4 * i + 1], o[n][m][4 * i + 2], o[n][m][4 * i + 3]};
      if (half == 0) {
        part_stats(p, at, D)[0] = top;
        part_stats(p, at, D)[1] = total;
      }
    }
  }
}

// Joins the parts of the rows of cut units: D / 4 lanes a row.
constexpr int kJoinThreads = 512;
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
    attention_prompt_join_kernel(const AttentionArgs p, int few, int cus, int most_splits) {
  constexpr int kRows = Shape<D>::kRows, kLanes = D / 4, kSlices = kRows * kLanes / kJoinThreads;
  const int lane = threadIdx.x & 63, slice = blockIdx.x % kSlices, cut = blockIdx.x / kSlices;
  const Cut c = cut_units(p, few, kRows, cus, most_splits, lane);
  const int unit = c.whole + cut;
  if (unit >= c.units) return;
  const RowTile where = find_row_tile(p, few, kRows, unit / p.cache.heads, lane);
  const Sequence s = sequence(p, where.seq);
  const int r = slice * (kJoinThreads / kLanes) + int(threadIdx.x) / kLanes;
  const int channel = threadIdx.x % kLanes * 4;
  const int row = (where.tiles - 1 - where.tile) * kRows + r;
  if (row >= s.rows) return;
  const int64_t first = int64_t(cut) * c.splits * kRows + r;
  float top = kLowest, total = 0;
  f32x4 x = {0, 0, 0, 0};
  // Parts i .. i + n - 1, on their way together; past the last they are that one again, and count 0.
  auto add = [&](int i, auto n) {
    f32x2 stats[n];
    f32x4 sums[n];
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const int64_t at = first + int64_t(min(i + j, c.splits - 1)) * kRows;
      stats[j] = *reinterpret_cast<const f32x2*>(part_stats(p, at, D));
      sums[j] = *reinterpret_cast<const f32x4*>(part_sums(p, at, D) + channel);
    }
    float most = top;
#pragma unroll
    for (int j = 0; j < n; ++j) most = fmaxf(most, stats[j][0]);
    const float old = __builtin_amdgcn_exp2f(top - most);
    top = most;
    total *= old;
    x *= old;
#pragma unroll
    for (int j = 0; j < n; ++j)
      if (i + j < c.splits) {
        const float factor = __builtin_amdgcn_exp2f(stats[j][0] - most);
        total += stats[j][1] * factor;
        x += sums[j] * factor;
      }
  };
  int i = 0;
  for (; i + 8 <= c.splits; i += 8) add(i, std::integral_constant<int, 8>());
  for (; i < c.splits; i += 2) add(i, std::integral_constant<int, 2>());
  write_row4(p, D, s.q_begin, row, unit % p.cache.heads, channel, x, top, total);
}

template <int D>
hipError_t launch_prompt(const AttentionArgs& args, int few, hipStream_t stream) {
  using S = Shape<D>;
  const int found = device_cu_count(), cus = found > 0 && found <= 256 ? found : 256;
  static_assert(256 * S::kRows <= kAttentionWorkspaceRows, "one part a CU");
  const int64_t units =
      prompt_units(args.tokens, args.seqs, args.group, args.max_q, args.cache.heads);
  // Cut into parts of four tiles or more. After many rounds the last one counts for little, and
  // the last units of prompts without a context before them are short by themselves.
  const int64_t longest = int64_t(args.table_width) << args.cache.page_shift;
  const bool windowed = args.window && int64_t(args.window) + args.max_q < longest;
  const int64_t seen = windowed ? args.window + args.max_q : longest;
  const int64_t rounds = windowed || longest >= 2 * int64_t(args.max_q) ? 8 : 1;
  int64_t splits = units <= rounds * cus ? seen / (4 * S::kTokens) : 1;
  if (splits > cus) splits = cus;
  if (splits < 1) splits = 1;
  const int64_t grid = units + (splits > 1 ? cus : 0);
  attention_prompt_kernel<D>
      <<<uint32_t(grid), S::kThreads, 0, stream>>>(args, few, cus, int(splits));
  if (splits == 1) return hipGetLastError();
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  // A unit that is cut has two parts or more.
  constexpr int kSlices = S::kRows * (D / 4) / kJoinThreads;
  attention_prompt_join_kernel<D>
      <<<uint32_t(cus / 2 * kSlices), kJoinThreads, 0, stream>>>(args, few, cus, int(splits));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_prompt(const AttentionArgs& args, int dim, int few, hipStream_t stream) {
  switch (dim) {
    case 64: return launch_prompt<64>(args, few, stream);
    case 128: return launch_prompt<128>(args, few, stream);
    default: return launch_prompt<256>(args, few, stream);
  }
}

}  // namespace ci8
