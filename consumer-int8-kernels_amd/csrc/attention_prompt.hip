// attention_fp4 for many query rows a sequence (include/consumer_int8_attention.h): prompts, and
// chunks of them behind a context.
//
// The mathematics and the order of operands are attention_split.hip's, with 32 x 32 x 16 MFMAs:
// S^T = K Q^T leaves a row's scores in the registers of its column's two lanes, where they are
// weighted and become the operand of O^T += V^T P^T without an exchange. Rows are (token, query
// head of one key head) pairs, 256 a workgroup, so that heads that share a key head share its
// tiles. Four operations a score and channel: bound by the MFMA rate, then by the softmax's
// vector instructions (about five a score) and by LDS reads (each wave reads every tile). So a
// wave takes 64 rows at D <= 128 (half the LDS reads of 32), one wave a SIMD with its 512
// registers, and the scores of the next tile are on the matrix unit while the vector unit
// weighs those of this one.
//
// Tiles of keys and values are converted to BF16 once a workgroup, on their way into LDS: global
// loads run two tiles ahead, one barrier a tile.
#include "attention_device.h"
#include "launch.h"

namespace ci8 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Rows of a workgroup in tiles of 32, its waves, and tokens of a tile.
template <int D>
struct Shape {
  static constexpr int kTiles = 1;  // of a wave
  static constexpr int kWaves = D <= 128 ? 8 : 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRows = 32 * kTiles * kWaves;
  static constexpr int kTokens = D == 64 ? 128 : D == 128 ? 64 : 32;
  static constexpr int kBlocks = D / kFp4Block;
  // Byte pitches of LDS rows: reads of 8 lanes' 16 bytes, and of 4 rows' 32 bytes transposed,
  // fall on different banks.
  static constexpr int kKeyPitch = 2 * D + 16, kValuePitch = 2 * D + 32;
  static constexpr int kKeyBytes = kTokens * kKeyPitch, kValueBytes = kTokens * kValuePitch;
  static constexpr int kPacks = 2 * kTokens * kBlocks / kThreads;  // 16 bytes of codes a thread
  static_assert(2 * kTokens * kBlocks % kThreads == 0);
};

// Row tiles of a sequence that this kernel has.
__device__ __forceinline__ int row_tiles(const Sequence& s, int few, int rows) {
  return s.rows <= few ? 0 : (s.rows + rows - 1) / rows;
}

// Which sequence and row tile: `index` counts all sequences' tiles.
struct RowTile {
  int seq, tile, tiles;  // seq < 0: past the last
};
__device__ __forceinline__ RowTile find_row_tile(const AttentionArgs& p, int few, int rows,
                                                 int index, int lane) {
  for (int base = 0; base < p.seqs; base += 64) {
    int n = 0;
    if (base + lane < p.seqs) n = row_tiles(sequence(p, base + lane), few, rows);
    const int sum = wave_scan(n, lane);
    const uint64_t hit = __ballot(sum > index);
    if (hit) {
      const int which = __builtin_ctzll(hit);
      const int tiles = uniform(__shfl(n, which, 64));
      return {base + which, index - (uniform(__shfl(sum, which, 64)) - tiles), tiles};
    }
    index -= uniform(__shfl(sum, 63, 64));
  }
  return {-1, 0, 0};
}

// Parts of the workspace: [unit][split][row][D] and the statistics after them.
__device__ __forceinline__ float* part_sums(const AttentionArgs& p, int64_t row, int dim) {
  return p.workspace + row * dim;
}
__device__ __forceinline__ float* part_stats(const AttentionArgs& p, int64_t row, int dim) {
  return p.workspace + int64_t(kAttentionWorkspaceRows) * dim + row * 2;
}

template <int D>
__global__ void __launch_bounds__(Shape<D>::kThreads)
    attention_prompt_kernel(const AttentionArgs p, int few, int splits) {
  using S = Shape<D>;
  constexpr int kTokens = S::kTokens, kTiles = S::kTiles, kHalves = kTokens / 32;
  constexpr int kSteps = D / 16, kChannels = D / 32;
  // Keys of tile t are read in the steps of tiles t - 1 and t, values in that of t.
  __shared__ __align__(16) char keys[3][S::kKeyBytes];
  __shared__ __align__(16) char values[2][S::kValueBytes];
  __shared__ uint32_t there_words[3][kTokens / 16];       // whether 16 tokens' page is
  __shared__ uint8_t poison[2][kTokens][S::kBlocks];      // NaN blocks of edge tiles
  __shared__ int poisoned[2];                             // the last such tile that has any

  const int thread = threadIdx.x, lane = thread & 63, wave = uniform(thread >> 6);
  const int column = lane & 31, half = lane >> 5;
  const int heads = p.cache.heads;
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits;
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
    const int n = max(t_end - t_begin, 0), part = (n + splits - 1) / splits;
    const int end = t_end;
    t_begin = min(t_begin + split * part, end);
    t_end = min(t_begin + part, end);
  }

  // The lane's rows and their tokens [low, high).
  int row_low[kTiles], row_high[kTiles];
  u32x4 q[kTiles][kSteps];
  const int wave_row = row0 + wave * 32 * kTiles;
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int row = wave_row + 32 * n + column;
    const bool live = row < s.rows;
    const int query = live ? row / p.group : 0;
    row_high[n] = live ? s.shift + query + 1 : 0;
    row_low[n] = p.window ? max(row_high[n] - p.window, 0) : 0;
    const uint16_t* src = p.q.data + int64_t(s.q_begin + query) * p.q.token_stride +
                          int64_t(kv_head * p.group + (live ? row % p.group : 0)) * p.q.head_stride;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
      q[n][j] = *reinterpret_cast<const u32x4*>(src + 16 * j + 8 * half);
  }
  // Tokens that all, or any, of the wave's live rows attend to.
  const int wave_last = min(wave_row + 32 * kTiles - 1, s.rows - 1);
  const bool wave_live = wave_row < s.rows;
  const int all_high = wave_live ? s.shift + wave_row / p.group + 1 : 0;
  const int any_high = wave_live ? s.shift + wave_last / p.group + 1 : 0;
  const int all_low = p.window ? max(any_high - p.window, 0) : 0;

  f32x16 o[kTiles][kChannels];
  float reference[kTiles], sum[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
#pragma unroll
    for (int m = 0; m < kChannels; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][m][i] = 0;
    reference[n] = kLowest;
    sum[n] = 0;
  }

  // Staging. Pack c of a thread is 32 channels of one token, of the keys first, then of the
  // values. `page` is loaded a tile ahead of the codes, these a tile ahead of their use.
  constexpr int kPerTile = kTokens * S::kBlocks;
  struct Staged {
    u32x4 codes;
    uint32_t scale;
    int page;
  };
  Staged staged[S::kPacks];
  auto is_value = [&](int c) __attribute__((always_inline)) { return c * S::kThreads + thread >= kPerTile; };
  auto token_of = [&](int c) __attribute__((always_inline)) { return (c * S::kThreads + thread) % kPerTile / S::kBlocks; };
  auto block_of = [&](int c) __attribute__((always_inline)) { return thread % S::kBlocks; };
  auto page_of = [&](int t, int c) __attribute__((always_inline)) {
    const int token = t * kTokens + token_of(c);
    int page = -1;
    if (t < t_end && token < s.context)
      page = p.page_table[int64_t(where.seq) * p.table_width + (token >> p.cache.page_shift)];
    return uint32_t(page) < uint32_t(p.cache.pages) ? page : -1;
  };
  int next_page[S::kPacks];
  // Tiles of the keys and of the values.
  auto load_pages = [&](int tk, int tv) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) next_page[c] = page_of(is_value(c) ? tv : tk, c);
  };
  auto load_codes = [&](int tk, int tv) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) {
      const int t = is_value(c) ? tv : tk;
      staged[c].page = next_page[c];
      staged[c].codes = u32x4{0, 0, 0, 0};
      staged[c].scale = 0;
      if (staged[c].page >= 0) {
        const Fp4Rows& rows = is_value(c) ? p.cache.v : p.cache.k;
        const int64_t row = (int64_t(kv_head) << p.cache.page_shift) +
                            ((t * kTokens + token_of(c)) & ((1 << p.cache.page_shift) - 1));
        staged[c].codes = *reinterpret_cast<const u32x4*>(
            rows.codes + staged[c].page * rows.code_stride + row * (D / 2) + 16 * block_of(c));
        staged[c].scale = rows.scales[staged[c].page * rows.scale_stride + row * S::kBlocks + block_of(c)];
      }
    }
  };
  auto edge_tile = [&](int t) __attribute__((always_inline)) {
    return (t + 1) * kTokens > first_high || t * kTokens < last_low;
  };
  auto store_tiles = [&](int tk, int tv) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::kPacks; ++c) {
      const int token = token_of(c), block = block_of(c);
      const bool value = is_value(c);
      const int t = value ? tv : tk, buffer = value ? t & 1 : t % 3;
      if (t >= t_end) continue;
      Staged x = staged[c];
      if (value && edge_tile(t)) {
        const bool nan = x.scale >= 253;
        poison[buffer][token][block] = nan;
        if (nan) {
          poisoned[buffer] = t;
          x.codes = u32x4{0, 0, 0, 0};
          x.scale = 0;
        }
      }
      if (!value && block == 0 && token % 16 == 0) there_words[buffer][token / 16] = x.page >= 0;
      char* to = value ? values[buffer] + token * S::kValuePitch : keys[buffer] + token * S::kKeyPitch;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<u32x4*>(to + 64 * block + 16 * j) =
            fp4_to_bf16x8(x.codes[j], fp4_scale(x.scale));
    }
  };

  // Half b of tile t is 32 tokens; its scores are computed while the half before is weighed.
  auto multiply = [&](int t, int b, f32x16(&score)[kTiles], uint32_t& holes)
      __attribute__((always_inline)) {
    const char* from = keys[t % 3] + (32 * b + column) * S::kKeyPitch + 16 * half;
    holes = (there_words[t % 3][2 * b] ? 0u : 1u) | (there_words[t % 3][2 * b + 1] ? 0u : 2u);
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) score[n][i] = 0;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(from + 32 * j);
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
        score[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, q[n][j]), score[n], 0, 0, 0);
    }
  };

  u32x4 weights[kTiles][2];
  auto weigh = [&](int first, f32x16(&score)[kTiles], uint32_t holes)
      __attribute__((always_inline)) {
    const bool edge = first + 32 > all_high || first < all_low || holes;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) score[n][i] *= p.scale_log2;
      if (edge) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 8 * (i / 4) + i % 4, token = first + at + 4 * half;
          const bool hidden =
              (token < row_low[n]) | (token >= row_high[n]) | ((holes >> (at / 16) & 1) != 0);
          score[n][i] = hidden ? -__builtin_inff() : score[n][i];
        }
      }
      float most = kLowest;
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, score[n][i]);
      if (__any(most > reference[n] + kSlack)) {
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        most = fmaxf(most, reference[n]);
        const float factor = __builtin_amdgcn_exp2f(reference[n] - most);
        reference[n] = most;
        sum[n] *= factor;
#pragma unroll
        for (int m = 0; m < kChannels; ++m) o[n][m] *= factor;
      }
      float total[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        score[n][i] = __builtin_amdgcn_exp2f(score[n][i] - reference[n]);
        total[i % 2] += score[n][i];
      }
      sum[n] += total[0] + total[1];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          weights[n][c][i] = pack_bf16x2(score[n][8 * c + 2 * i], score[n][8 * c + 2 * i + 1]);
    }
  };
  auto add_values = [&](int t, int half_tile) __attribute__((always_inline)) {
    const char* from = values[t & 1] +
                       (32 * half_tile + 4 * half + lane % 16 / 4) * S::kValuePitch +
                       (16 * (lane / 16 % 2) + 4 * (lane % 4)) * 2;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < kChannels; ++m) {
        const u32x2 a = lds_read_transposed(from + 16 * c * S::kValuePitch + 64 * m);
        const u32x2 b = lds_read_transposed(from + (16 * c + 8) * S::kValuePitch + 64 * m);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          o[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]}),
              __builtin_bit_cast(bf16x8, weights[n][c]), o[n][m], 0, 0, 0);
      }
  };
  // NaN blocks of an edge tile's values stand as zeros; rows that see their token get the NaN.
  auto add_poison = [&](int t) __attribute__((always_inline)) {
    for (int token = 0; token < kTokens; ++token)
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
        if (poison[t & 1][token][m]) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
            if (t * kTokens + token >= row_low[n] && t * kTokens + token < row_high[n])
              o[n][m] += __builtin_nanf("");
        }
  };

  f32x16 scores[2][kTiles];
  uint32_t holes[2];
  if (thread < 2) poisoned[thread] = -1;
  __syncthreads();
  if (t_begin < t_end) {
    // Keys run a tile ahead of values.
    load_pages(t_begin, t_end);
    load_codes(t_begin, t_end);
    load_pages(t_begin + 1, t_begin);
    store_tiles(t_begin, t_end);
    load_codes(t_begin + 1, t_begin);
    load_pages(t_begin + 2, t_begin + 1);
    store_tiles(t_begin + 1, t_begin);
    load_codes(t_begin + 2, t_begin + 1);
    load_pages(t_begin + 3, t_begin + 2);
    __syncthreads();
    multiply(t_begin, 0, scores[0], holes[0]);
    __syncthreads();
  }
  // Scores alternate between two sets of registers; tiles of one half are unrolled in pairs.
  auto step = [&](int t, auto parity) __attribute__((always_inline)) {
    constexpr int first = kHalves % 2 == 0 ? 0 : decltype(parity)::value;
#pragma unroll
    for (int b = 0; b < kHalves; ++b) {
      const int now = (first + b) % 2, after = 1 - now;
      if (b + 1 < kHalves)
        multiply(t, b + 1, scores[after], holes[after]);
      else if (t + 1 < t_end)
        multiply(t + 1, 0, scores[after], holes[after]);
      weigh(t * kTokens + 32 * b, scores[now], holes[now]);
      if (b == 0) {
        store_tiles(t + 2, t + 1);
        load_codes(t + 3, t + 2);
        load_pages(t + 4, t + 3);
      }
      add_values(t, b);
    }
    if (edge_tile(t) && poisoned[t & 1] == t) add_poison(t);
    __syncthreads();
  };
  for (int t = t_begin; t < t_end;) {
    step(t, std::integral_constant<int, 0>{});
    ++t;
    if (kHalves % 2 == 0) continue;
    if (t >= t_end) break;
    step(t, std::integral_constant<int, 1>{});
    ++t;
  }

  // A row's two lanes hold the sums of their own tokens.
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const float total = sum[n] + __shfl_xor(sum[n], 32, 64);
    const int row = wave_row + 32 * n + column;
    if (row >= s.rows) continue;
    if (splits == 1) {
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = {o[n][m][4 * i], o[n][m][4 * i + 1], o[n][m][4 * i + 2], o[n][m][4 * i + 3]};
          write_row4(p, D, s.q_begin, row, kv_head, 32 * m + 8 * i + 4 * half, x, reference[n], total);
        }
    } else {
      const int64_t at = int64_t(blockIdx.x) * S::kRows + (row - row0);
#pragma unroll
      for (int m = 0; m < kChannels; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(part_sums(p, at, D) + 32 * m + 8 * i + 4 * half) =
              f32x4{o[n][m][4 * i], o[n][m][4 * i + 1], o[n][m][4 * i + 2], o[n][m][4 * i + 3]};
      if (half == 0) {
        part_stats(p, at, D)[0] = reference[n];
        part_stats(p, at, D)[1] = total;
      }
    }
  }
}

// Joins the splits of each row: D / 4 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) attention_prompt_join_kernel(const AttentionArgs p, int few,
                                                                    int splits) {
  constexpr int kRows = Shape<D>::kRows, kLanes = D / 4, kSlices = kRows * kLanes / 256;
  const int lane = threadIdx.x & 63, slice = blockIdx.x % kSlices, unit = blockIdx.x / kSlices;
  const RowTile where = find_row_tile(p, few, kRows, unit / p.cache.heads, lane);
  if (where.seq < 0) return;
  const Sequence s = sequence(p, where.seq);
  const int r = slice * (256 / kLanes) + int(threadIdx.x) / kLanes;
  const int channel = threadIdx.x % kLanes * 4;
  const int row = (where.tiles - 1 - where.tile) * kRows + r;
  if (row >= s.rows) return;
  const int64_t first = int64_t(unit) * splits * kRows + r;
  float top = kLowest, total = 0;
  for (int i = 0; i < splits; ++i) top = fmaxf(top, part_stats(p, first + int64_t(i) * kRows, D)[0]);
  f32x4 x = {0, 0, 0, 0};
  for (int i = 0; i < splits; ++i) {
    const int64_t at = first + int64_t(i) * kRows;
    const float factor = __builtin_amdgcn_exp2f(part_stats(p, at, D)[0] - top);
    total += part_stats(p, at, D)[1] * factor;
    x += *reinterpret_cast<const f32x4*>(part_sums(p, at, D) + channel) * factor;
  }
  write_row4(p, D, s.q_begin, row, unit % p.cache.heads, channel, x, top, total);
}

template <int D>
hipError_t launch_prompt(const AttentionArgs& args, int few, hipStream_t stream) {
  using S = Shape<D>;
  const int found = device_cu_count(), cus = found > 0 ? found : 256;
  // Row tiles of all sequences, at most: each but its last is full.
  const int64_t rows = int64_t(args.tokens) * args.group;
  const int64_t each = (int64_t(args.max_q) * args.group + S::kRows - 1) / S::kRows;
  const int64_t bound = rows / S::kRows + args.seqs;
  const int64_t units = (bound < each * args.seqs ? bound : each * args.seqs) * args.cache.heads;
  // Contexts are cut where row tiles alone leave CUs idle, into parts of four tiles or more.
  const int64_t longest = int64_t(args.table_width) << args.cache.page_shift;
  const int64_t seen = args.window && args.window + args.max_q < longest ? args.window + args.max_q : longest;
  int64_t splits = cus / units;
  if (splits > seen / (4 * S::kTokens)) splits = seen / (4 * S::kTokens);
  if (splits < 1) splits = 1;
  if (units * splits * S::kRows > kAttentionWorkspaceRows && splits > 1)
    splits = kAttentionWorkspaceRows / (units * S::kRows);
  attention_prompt_kernel<D><<<uint32_t(units * splits), S::kThreads, 0, stream>>>(args, few, int(splits));
  if (splits == 1) return hipGetLastError();
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  attention_prompt_join_kernel<D>
      <<<uint32_t(units * (S::kRows * (D / 4) / 256)), 256, 0, stream>>>(args, few, int(splits));
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
