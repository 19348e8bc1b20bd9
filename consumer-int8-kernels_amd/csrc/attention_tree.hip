// attention_fp4_tree for more than a few rows a sequence (include/consumer_int8_drafts.h): the tens to
// hundreds of rows that the drafted tokens of a tree make with the query heads of a key head.
//
// The mathematics is attention_split.hip's, a wave works alone on 32 tokens at a time as there, and
// runs, parts and their joints are the same (attention_runs.h). A block is 64 rows, in two tiles of 32 (32
// rows in one at 256 channels), with 32 x 32 x 16 MFMAs:
//
//   S^T = K Q^T      K as the row operand straight from its codes: lane l holds token l % 32 and half
//                    l / 32 of the channels, eight a step; the contraction takes the channels in
//                    that order for K and Q alike.
//   O^T += V^T P^T   the S^T result layout (lane: row l % 32, tokens 8 (i/4) + 4 (l/32) + i % 4) is the
//                    operand layout of P^T; V is converted in the lane that loads it, stored to the
//                    wave's own LDS tile and read transposed with the tokens in that order.
//
// Two waves a SIMD, eight a workgroup, which share the queries in LDS; the sums of the rows take half of
// the registers. Every block of a key head reads and converts its tokens anew, from the caches between
// it and HBM: what bounds it is the issue of a SIMD's two waves. 64 rows of 128 channels take a wave 3600
// clocks a tile, 1024 of them MFMAs; over a long call vector instructions are half of all clocks, MFMAs a
// third. Larger blocks convert less, but four tiles of rows at 512 registers a wave took longer (one wave a
// SIMD has nobody to hide behind), and so did workgroups that share converted tokens through LDS, with
// their barriers.
//
// Queries of S and values of O are read from LDS some products ahead, with the compiler kept from
// moving the reads back together; addresses are computed anew in each tile from one number for each kind,
// since registers held for all of them through the loop were spilled.
//
// What a row sees of 32 tokens is one word of bits (tree_sees), in tiles on the edge only.
//
// Weights are rounded to BF16 for the second product, and their sum is of the FP32 weights, as in
// attention_split.hip and for its reason: outputs are 0.0019 to 0.0021 from 64 bits where FP32 weights give
// 0.0017, which is the outputs' own rounding.
//
// Measured, us, and in turn with it the split kernel in blocks of 64 rows: 8 x 64 tokens behind up to 16000
// of 40 query and 8 key heads of 128 151 and 169, 60 % of the rate that a large product of matrices reaches
// (workgroups that share converted tokens took 228 when the blocks took 182); 16 x 16 tokens behind up to
// 8000 of 32 and 8 heads 49 and 53; 32 x 11 of 28 and 4 heads with a window of 1024 21 and 26. 4 x 26 behind
// up to 131071 of 24 and 4 heads of 256 348, and workgroups that share converted tokens 347.
#include "attention_runs.h"
#include "launch.h"

namespace ci8 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int D>
struct TreeShape {
  static constexpr int kTiles = D == 256 ? 1 : 2, kRows = 32 * kTiles;  // of a block
  static_assert(kRows == tree_rows(D));
  static constexpr int kWaves = 8, kThreads = 64 * kWaves;
  static constexpr int kSteps = D / 16;       // MFMAs over the channels; 8 channels of a lane each
  static constexpr int kTilesOut = D / 32;    // of channels
  static constexpr int kBlocks = D / 64;      // scale blocks of a lane
  static constexpr int kScaleBytes = D / kFp4Block;
  static constexpr int kValueBytes = kTokens * 2 * D;
  static constexpr int kJoined = D < 128 ? D : 128;  // channels that waves join at once
  static constexpr int kJoinPitch = kJoined + 4;     // floats
  static constexpr int kJoinBytes = 32 * kJoinPitch * 4;
  static constexpr int kWaveBytes = kValueBytes > kJoinBytes ? kValueBytes : kJoinBytes;
};

// Codes and scales of 32 tokens' rows: this lane's token and half of its channels. Scales stay the words
// that hold them until they are used.
template <int D>
struct TreeRaw {
  uint32_t codes[D / 16];
  uint32_t scales;
};

// A value of which nothing is computed ahead of a loop, to be held through it.
__device__ __forceinline__ uint32_t anew(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

template <int D, bool kSplit>
__global__ void __launch_bounds__(TreeShape<D>::kThreads, 2)
    attention_tree_kernel(const AttentionArgs, int most, int most_blocks, int min_quota,
                          bool by_context, bool apart) {
  using S = TreeShape<D>;
  constexpr int kTiles = S::kTiles, kWaves = S::kWaves, kSteps = S::kSteps;
  constexpr int kAhead = 4, kValuesAhead = 2;
  __shared__ __align__(256) char shared[kWaves * S::kWaveBytes];
  __shared__ u32x4 queries[kTiles * kSteps * 64];
  __shared__ float tops[kWaves][S::kRows], sums[kWaves][S::kRows];
  __shared__ uint64_t tree[64];  // what each query sees of the tree, bit a for query a

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 31, half = lane >> 5;

  // Workgroups of an XCD take runs that follow each other: blocks of one key head, which read the same
  // tokens, then share an L2.
  const int group = gridDim.x % 8 ? blockIdx.x : blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  const int begin = apart ? 0 : kTreeBegin;
  Run run;
  Place place;
  if constexpr (kSplit) {
    const AttentionArgs& p = arguments();
    Counted counted = count_costs(p, most, S::kRows, begin, lane, 0);
    int64_t total = all_costs(p, most, S::kRows, begin, lane, counted);
    run.quota = uniform(max((total + gridDim.x - 1) / gridDim.x, int64_t(min_quota)));
    if (apart) {
      int quota = int(run.quota), parts;
      for (;; quota += quota / 64 + 1) {
        parts = (counted.cost + quota - 1) / quota;
        if (wave_sum(counted.blocks * parts) * p.cache.heads <= int(gridDim.x)) break;
      }
      counted.cost = parts * quota;
      counted.sum = wave_scan(counted.blocks * counted.cost);
      total = int64_t(at_lane(counted.sum, 63)) * p.cache.heads;
      run.quota = quota;
    }
    run.begin = group * run.quota;
    run.end = min(run.begin + run.quota, total);
    if (!by_context && threadIdx.x == 0) joints<D>(p)[group].parts = 0;
    if (run.begin >= total) return;
    place = find_place(p, most, S::kRows, begin, lane, run.begin, counted);
  } else {
    const AttentionArgs& p = arguments();
    place.block = group % most_blocks;
    place.head = group / most_blocks % p.cache.heads;
    place.seq = group / most_blocks / p.cache.heads;
    const Sequence s = sequence(p, place.seq);
    place.blocks = uniform(row_blocks(s, most, S::kRows));
    if (place.block >= place.blocks) return;
    place.at = 0;
    place.cost = uniform(block_tiles(s));
    run = {0, place.cost, place.cost};
  }
  // Where this lane's codes and scales of a token's row start, the bytes of its scales in their word,
  // and its places in the LDS tile: pieces of 8 channels of a token's row are XORed by the token, so
  // that both the stores of 8 tokens and transposed reads fall on different banks.
  const uint32_t page_row = column & ((1 << arguments().cache.page_shift) - 1);
  const uint32_t code_at = page_row * (D / 2) + half * (D / 4);
  const uint32_t scale_at = (page_row * S::kScaleBytes + half * S::kBlocks) & ~3u;
  char* const tile = shared + wave * S::kWaveBytes;
  uint32_t store_at, read_at, scale_byte;  // the last: of the lane's first scale in its word
  {
    const uint32_t lane = threadIdx.x & 63, half = lane / 32;
    const uint32_t token = lane % 32, row = 4 * half + lane % 16 / 4;
    store_at = token * (2 * D) + ((half * D) ^ (16 * (token % 8)));
    read_at = row * (2 * D) + 64 * half + 16 * ((2 * (lane / 16 % 2) + lane % 4 / 2) ^ (row & 3)) +
              lane % 2 * 8;
    scale_byte = (token * S::kScaleBytes + half * S::kBlocks) % 4;
  }

  for (int64_t at = run.begin; at < run.end;) {
    const int seq = place.seq, kv_head = place.head;
    const AttentionArgs& p = arguments();
    const int page_mask = (1 << p.cache.page_shift) - 1;
    const Sequence s = sequence(p, seq);
    const int row0 = place.block * S::kRows, rows = min(s.rows - row0, S::kRows);
    const int take = int(min(int64_t(place.cost - place.at), run.end - at));
    // The run's share of the context's cost is its share of the tiles.
    const int tiles = block_tiles(s);
    const float share = float(tiles) / float(place.cost);
    auto tile_at = [&](int cost) {
      return s.first_tile(kTokens) +
             uniform(cost == place.cost ? tiles : min(int(float(cost) * share), tiles));
    };
    const int t_begin = tile_at(place.at), t_end = tile_at(place.at + take);

    // This wave's tiles are t_begin + wave, + kWaves, ...; lane 2i + h holds the page of half h of the
    // i-th, for 32 of them. Pages outside the cache are page 0 and have no bit in `in_cache`.
    int page_of = 0;
    uint64_t in_cache = 0;
    auto load_pages = [&](int first) {
      const int lane = int(anew(threadIdx.x & 63));
      const int t = first + (lane >> 1) * kWaves;
      const int token = t * kTokens + 16 * (lane & 1);
      int page = -1;
      if (t < t_end && token < s.context)
        page = p.page_table[int64_t(seq) * p.table_width + (token >> p.cache.page_shift)];
      const bool there = uint32_t(page) < uint32_t(p.cache.pages);
      in_cache = __ballot(there);
      page_of = there ? page : 0;
    };
    const int t_first = t_begin + wave;
    if (t_first < t_end) load_pages(t_first);
    const bool some_tree = p.window || t_end * kTokens > s.shift;
    int parent = -1;
    if (some_tree) parent = tree_parent(p, s, lane);

    // The lane's rows, and the tokens [low, high) that each attends to. Rows that are not there repeat
    // one that is; their results go nowhere.
    int low[kTiles], high[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const int row = row0 + 32 * n + column;
      high[n] = row < s.rows ? s.shift + row / p.group + 1 : 0;
      low[n] = 0;
    }
    __syncthreads();  // the last queries are read
#pragma unroll 1
    for (int i = wave; i < kTiles * kSteps; i += kWaves) {
      const int lane = int(anew(threadIdx.x & 63)), row = row0 + i / kSteps * 32 + lane % 32;
      const bool live = row < s.rows;
      const uint16_t* src =
          p.q.data + int64_t(s.q_begin + (live ? row / p.group : 0)) * p.q.token_stride +
          int64_t(kv_head * p.group + (live ? row % p.group : 0)) * p.q.head_stride;
      queries[i * 64 + lane] =
          *reinterpret_cast<const u32x4*>(src + lane / 32 * (D / 2) + i % kSteps * 8) ^ p.q_sign;
    }

    const int64_t head_row = int64_t(kv_head) << p.cache.page_shift;
    // Tile t, the i-th of those looked up: of one page, or of two of 16 tokens.
    const bool one_page = page_mask >= 31;
    auto load = [&](TreeRaw<D>& raw, const Fp4Rows& rows, int t, int i) __attribute__((always_inline)) {
      const int64_t row = head_row + (uint32_t(t * kTokens) & page_mask);
      const uint8_t* const codes = rows.codes + row * (D / 2);
      const uint8_t* const scales = rows.scales + row * S::kScaleBytes;
      auto fill = [&](uint64_t code, uint64_t scale) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(codes + code + code_at + 16 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) raw.codes[4 * j + i] = w[i];
        }
        raw.scales = *reinterpret_cast<const uint32_t*>(scales + scale + scale_at);
      };
      const uint64_t page = uint32_t(__builtin_amdgcn_readlane(page_of, 2 * i));
      const uint64_t code = page * rows.code_stride, scale = page * rows.scale_stride;
      if (one_page) {
        fill(code, scale);
      } else {
        const uint64_t other = uint32_t(__builtin_amdgcn_readlane(page_of, 2 * i + 1));
        const uint64_t code2 = other * rows.code_stride, scale2 = other * rows.scale_stride;
        fill(column < 16 ? code : code2, column < 16 ? scale : scale2);
      }
    };
    // Eight channels of step j, with the lane's first scale at `byte` of its word.
    auto converted = [&](const TreeRaw<D>& raw, int j, uint32_t byte) __attribute__((always_inline)) {
      return fp4_to_bf16x8(raw.codes[j], fp4_scale_in(raw.scales, fp4_scale_turn(byte + j / 4)));
    };

    f32x16 o[kTiles][S::kTilesOut];
    float reference[kTiles], sum[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int m = 0; m < S::kTilesOut; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][m][i] = 0;
      reference[n] = kLowest;
      sum[n] = 0;
    }

    // Keys and values of a tile each take the registers of the last as soon as those are used. After the
    // wave's last tile the loads go on with that one again: were they skipped, the waits for those before
    // would have to be for all.
    TreeRaw<D> k, v;
    int t = t_first, i = 0, there = 3;
    if (t < t_end) {
      load(k, p.cache.k, t, 0);
      load(v, p.cache.v, t, 0);
      there = int(in_cache & 3);
    }
    if (some_tree) {  // with the first tile on its way
      const uint64_t set = tree_ancestors(parent, lane);
      const int depth = __builtin_popcountll(set) - 1;
      tree[lane] = tree_seen(p, set);  // every wave the same
      wave_order();
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
        low[n] = tree_low(p, s, depth, max(high[n] - 1 - s.shift, 0) & 63);
    }
    __syncthreads();
    while (t < t_end) {
      const bool more = t + kWaves < t_end;
      const int t_next = more ? t + kWaves : t;
      if (more && ++i == 32) {
        load_pages(t_next);
        i = 0;
      }
      // Tiles that some row sees in part, or that are not whole.
      const bool edge = (t + 1) * kTokens > s.shift || t * kTokens < s.last_low || there != 3;
      // Two chains of products at least: one takes twice as long as the matrix unit.
      f32x16 x[2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[n][i] = 0;
      // Queries are read kAhead operands before their products.
      const u32x4* const mine = queries + anew(lane);
      constexpr int kProducts = kTiles * kSteps;
      u32x4 operand[kAhead];
      auto query = [&](int i) { return mine[(i % kTiles * kSteps + i / kTiles) * 64]; };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) operand[i] = query(i);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      bf16x8 key;
      const uint32_t key_byte = anew(scale_byte);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        if (i % kTiles == 0) key = __builtin_bit_cast(bf16x8, converted(k, i / kTiles, key_byte));
        x[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            key, __builtin_bit_cast(bf16x8, operand[i % kAhead]), x[i % 2], 0, 0, 0);
        if (i + kAhead < kProducts) operand[i % kAhead] = query(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (kTiles == 1) x[0] += x[1];
      load(k, p.cache.k, t_next, i);

      uint32_t poisoned = 0;
      if (edge) {
        const int half = int(anew(lane)) >> 5, column = int(anew(lane)) & 31;
        // Values of tokens past the context or of no page are zeros, and so are blocks that are
        // NaN, since some row may not see their token and its weight of 0 would not keep them out.
        const int token = t * kTokens + column;
        const bool real = (there >> (column / 16) & 1) && token < s.context;
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b) {
          const uint32_t shift = (anew(scale_byte) + b) * 8;
          if (!real || (v.scales >> shift & 0xFF) >= 253) {
            if (real) poisoned |= 1u << (half * S::kBlocks + b);
#pragma unroll
            for (int j = 0; j < 4; ++j) v.codes[4 * b + j] = 0;
            v.scales &= ~(0xFFu << shift);
          }
        }
        poisoned |= uint32_t(__shfl_xor(int(poisoned), 32, 64));
        const uint32_t pages = (there & 1 ? 0xFFFFu : 0) | (there & 2 ? 0xFFFF0000u : 0);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          const uint32_t sees =
              (tree_sees(tree, low[n], high[n], t * kTokens, s.shift) & pages) >> (4 * half);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[n][i] = sees >> (8 * (i / 4) + i % 4) & 1 ? x[n][i] : -__builtin_inff();
        }
      }
      wave_order();
      const uint32_t value_byte = anew(scale_byte), to = anew(store_at);
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        *reinterpret_cast<u32x4*>(tile + (to ^ (16 * j))) = converted(v, j, value_byte);
      wave_order();
      load(v, p.cache.v, t_next, i);
      // The first values' operands come while the scores are weighed.
      const uint32_t from = anew(read_at);
      auto value = [&](int i) {
        const char* at = tile + ((from ^ (64 * (i / 2))) + 16 * (i % 2) * (2 * D));
        const u32x2 a = lds_read_transposed(at), b = lds_read_transposed(at + 8 * (2 * D));
        return u32x4{a[0], a[1], b[0], b[1]};
      };
      u32x4 values[kValuesAhead];
#pragma unroll
      for (int i = 0; i < kValuesAhead; ++i) values[i] = value(i);

      float peak[kTiles];
      bool passes = false;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        peak[n] = x[n][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) peak[n] = fmaxf(peak[n], x[n][i]);
        peak[n] *= p.scale_log2;
        passes = passes || peak[n] > reference[n] + kSlack;
      }
      if (__any(passes)) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float m = fmaxf(peak[n], __shfl_xor(peak[n], 32, 64));
          m = m > reference[n] + kSlack ? m : reference[n];
          const float factor = __builtin_amdgcn_exp2f(reference[n] - m);
          reference[n] = m;
          sum[n] *= factor;
#pragma unroll
          for (int c = 0; c < S::kTilesOut; ++c) o[n][c] *= factor;
        }
      }
      u32x4 weights[kTiles][2];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        float total[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[n][i] = __builtin_amdgcn_exp2f(fmaf(x[n][i], p.scale_log2, -reference[n]));
          total[i % 2] += x[n][i];
        }
        sum[n] += total[0] + total[1];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            weights[n][c][i] = pack_bf16x2(x[n][8 * c + 2 * i], x[n][8 * c + 2 * i + 1]);
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2 * S::kTilesOut; ++i) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          o[n][i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, values[i % kValuesAhead]),
              __builtin_bit_cast(bf16x8, weights[n][i % 2]), o[n][i / 2], 0, 0, 0);
        if (i + kValuesAhead < 2 * S::kTilesOut)
          values[i % kValuesAhead] = value(i + kValuesAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (edge && __any(poisoned)) {
        for (int token = 0; token < kTokens; ++token) {
          const uint32_t blocks = uint32_t(__shfl(int(poisoned), token, 64));
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
            if (blocks && tree_sees(tree, low[n], high[n], t * kTokens, s.shift) >> token & 1) {
#pragma unroll
              for (int m = 0; m < S::kTilesOut; ++m)
                o[n][m] += blocks >> m & 1 ? __builtin_nanf("") : 0.f;
            }
        }
      }
      there = int(in_cache >> (2 * i) & 3);
      t += kWaves;
    }

    // Joins the waves: one tile of rows at a time through LDS. Lane numbers are taken anew, so that
    // nothing of this is computed ahead and held through the loop above.
    {
    const AttentionArgs& p = arguments();
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, column = lane & 31, half = lane >> 5;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      sum[n] += __shfl_xor(sum[n], 32, 64);
      if (half == 0) {
        tops[wave][32 * n + column] = reference[n];
        sums[wave][32 * n + column] = sum[n];
      }
    }
    __syncthreads();
    const bool whole = place.at == 0 && take == place.cost;
    const int part = 2 * group + (place.at == 0 ? 1 : 0);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float top = kLowest;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w][32 * n + column]);
      const float factor = __builtin_amdgcn_exp2f(reference[n] - top);
      float* join = reinterpret_cast<float*>(tile) + column * S::kJoinPitch + 4 * half;
#pragma unroll
      for (int first = 0; first < D; first += S::kJoined) {
#pragma unroll
        for (int m = 0; m < S::kJoined / 32; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x16& x = o[n][first / 32 + m];
            *reinterpret_cast<f32x4*>(join + 32 * m + 8 * i) =
                f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]} * factor;
          }
        __syncthreads();
        for (int i = thread; i < 32 * S::kJoined / 4; i += S::kThreads) {
          const int r = i / (S::kJoined / 4), row = 32 * n + r, channel = i % (S::kJoined / 4) * 4;
          if (row >= rows) continue;
          float all = kLowest, l = 0;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) all = fmaxf(all, tops[w][row]);
          f32x4 x = {0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            l += sums[w][row] * __builtin_amdgcn_exp2f(tops[w][row] - all);
            x += *reinterpret_cast<const f32x4*>(shared + w * S::kWaveBytes +
                                                 (r * S::kJoinPitch + channel) * 4);
          }
          if (!kSplit || whole) {
            write_row4(p, D, s.q_begin, row0 + row, kv_head, first + channel, x, all, l);
          } else {
            *reinterpret_cast<f32x4*>(part_sums<D, 2 * kTiles>(p, part) + row * D + first + channel) = x;
            if (first + channel == 0) {
              float* stats = part_stats<D, 2 * kTiles>(p, part) + row * 2;
              stats[0] = all;
              stats[1] = l;
            }
          }
        }
        __syncthreads();
      }
    }
    if (kSplit && place.at == 0 && (by_context || !whole) && threadIdx.x == 0) {
      const int64_t last = at + place.cost - 1;
      joints<D>(p)[by_context ? (seq * p.cache.heads + kv_head) * most_blocks + place.block
                              : group] = {
          whole ? 0 : int(last / run.quota) - group + 1, group, s.q_begin,
          row0, rows, kv_head};
    }
    }
    // On to the next block, key head or sequence.
    at += take;
    if (at < run.end) {
      place.at = 0;
      if (place.block + 1 < place.blocks) {
        ++place.block;
      } else if (place.block = 0; place.head + 1 < p.cache.heads) {
        ++place.head;
      } else {
        // More is left, so a later sequence has some.
        place.head = 0;
        do {
          ++place.seq;
          const Sequence next = sequence(p, place.seq);
          place.blocks = uniform(row_blocks(next, most, S::kRows));
          place.cost = uniform(block_tiles(next)) + begin;
        } while (place.blocks == 0 && place.seq + 1 < p.seqs);
      }
    }
  }
}

// Up to this many tiles of the longest context a workgroup takes a whole one of each block of rows, and
// up to twice as many if there are contexts for a third of the CUs. Whole and in equal runs with their
// joins, us: 49 rows of 28 and 4 heads of 128 behind up to 1100 tokens 18.8 and 19.5, 32 of them 20.3 and
// 32.0; behind up to 2000 26.7 and 22.0, 8 of them 26.7 and 23.4, of 182 rows 28.0 and 34.2, 32 of them
// 48.2 and 59.8.
constexpr int kWholeTreeTiles = 36;

template <int D>
hipError_t launch_tree(const AttentionArgs& args, hipStream_t stream) {
  using S = TreeShape<D>;
  const int64_t longest = (int64_t(args.table_width) << args.cache.page_shift) / kTokens;
  const int64_t span = args.window ? (int64_t(args.window) + args.max_q) / kTokens + 2 : longest;
  const int most = args.max_q * args.group;
  const int blocks = (most + S::kRows - 1) / S::kRows;
  const int64_t contexts = int64_t(args.seqs) * args.cache.heads * blocks;
  const int found = device_cu_count(), groups = found > 0 && found <= 256 ? found : 256;
  const bool few = 3 * contexts < groups;
  if ((longest < span ? longest : span) <= (few ? 1 : 2) * kWholeTreeTiles &&
      launch_fits(contexts, S::kThreads)) {
    attention_tree_kernel<D, false>
        <<<uint32_t(contexts), S::kThreads, 0, stream>>>(args, most, blocks, 0, false, false);
    return hipGetLastError();
  }
  static_assert(2 * 256 * S::kRows * 2 <= kAttentionWorkspaceRows * 2 - 2048 * 8,
                "parts, statistics and descriptions fit the workspace");
  const bool by_context = contexts <= groups;
  // With more than three workgroups a context, as in the split kernel. us, contexts apart and runs of all, by
  // contexts for 256 workgroups: 80 (10 x 16 tokens of 8 heads of 128) 36 and no less; 88 37 and 43, 128 49 and
  // 50; but 160 of 5 blocks 95 and 87, 192 69 and 62, 248 85 and 73; of 4 heads of 256, 5 blocks, 100 105 and
  // 102, 120 154 and 128.
  const bool apart = few && args.seqs <= 64;
  attention_tree_kernel<D, true><<<groups, S::kThreads, 0, stream>>>(
      args, most, blocks, 2 * S::kWaves, by_context, apart);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const bool many = groups > 16 * contexts;
  const auto join = many ? attention_join_kernel<D, 2 * S::kTiles, 1024>
                         : attention_join_kernel<D, 2 * S::kTiles, 512>;
  join<<<dim3(by_context ? uint32_t(contexts) : groups, D / kJoinChannels), many ? 1024 : 512, 0,
         stream>>>(args, most, blocks, groups, by_context);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_tree(const AttentionArgs& args, int dim, hipStream_t stream) {
  switch (dim) {
    case 64: return launch_tree<64>(args, stream);
    case 128: return launch_tree<128>(args, stream);
    default: return launch_tree<256>(args, stream);
  }
}

}  // namespace ci8
