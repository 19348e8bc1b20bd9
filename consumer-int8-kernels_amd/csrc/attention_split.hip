// attention_fp4 for few query rows a sequence (include/consumer_int8_attention.h): causal
// attention of BF16 queries over a paged cache of E2M1 values with power-of-two scales.
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp2(s_t - m),   s_t = q.k_t * scale * log2(e)
//
// in one pass with a running reference m. Rows are (token, query head of one key head) pairs,
// 16 or 32 at a time, so that the cache is read once for all heads that share it: bound by HBM, whose
// stream the conversions (half an instruction a value) and MFMAs have to stay under. A wave
// works alone on 32 tokens at a time, the next 32 on their way:
//
//   S^T = K Q^T      v_mfma_f32_16x16x32_bf16, K as the row operand: lane l holds token l % 16
//                    and the channels of its own scale block, 16 bytes of codes as they lie in
//                    the cache, converted by one instruction a pair. The contraction takes the
//                    channels in that order for K and Q alike.
//   O^T += V^T P^T   the S^T result layout (lane: row l % 16, tokens 4 (l/16) + i of each half)
//                    is already the operand layout of P^T; V is converted in the lane that
//                    loads it, stored to the wave's own LDS tile and read transposed
//                    (ds_read_b64_tr_b16) with the tokens in that order.
//
// The weights are rounded to BF16 for the second product, since BF16 is what its MFMA takes (FP32 weights
// would need a second BF16 product for what the first leaves, in a loop that runs close to HBM): 2^-8 of
// each at most, averaged over the tokens. Their sum is of the FP32 weights. Outputs are 0.0019 to 0.0022
// from 64 bits where FP32 weights give 0.0016 to 0.0017, most of it the outputs' own rounding.
//
// All statistics of a row sit in the lanes of its column. m moves only when a score passes it by
// 2^8 in weight, so most tiles exchange nothing between lanes and rescale nothing.
//
// Contexts differ and only the device knows them, so the work is cut there: all tiles of all
// sequences, key heads and blocks of rows are laid end to end, each context with what it costs to
// begin it, and each workgroup takes an equal run of them.
// A run that covers a whole context writes its output; parts of one go to the workspace, two
// at most a workgroup, and a second kernel joins them in a fixed order.
//
// Measured, of the cache's bytes: 64 contexts up to 32768 tokens, 64 query heads on 8 of 128, 257
// to 266 us, 5.4 to 5.6 TB/s (a stream of reads alone reaches 5.9 to 6.06); 32 up to 8000 40 us, 3.7
// TB/s with the join (5 us) and the way into the pipeline counted; one of 517 tokens 7.4 us, nearly all
// the launch.
#include "attention_device.h"
#include "attention_plan.h"
#include "launch.h"

namespace ci8 {
namespace {

constexpr int kTokens = 32;  // tokens a wave takes at once

// Keeps LDS accesses of a wave's lanes in program order; the LDS itself does.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int D>
struct Layout {
  // Channels a lane holds of a chunk: its own 16 bytes of codes (8 at D = 64).
  static constexpr int kChunk = D == 64 ? 16 : 32;
  static constexpr int kChunks = D / (4 * kChunk);
  static constexpr int kSteps = kChunk / 8;  // MFMA steps of a chunk
  static constexpr int kPitch = 2 * D + 32;  // bytes between token rows of the LDS tile
  static constexpr int kScaleBytes = D / kFp4Block;
};

// Codes and scales of 16 tokens' rows: this lane's token l % 16 and its chunks. Scales stay the
// words that hold them until they are used: bytes carried round a loop would be masked, and so
// waited for, at its end.
template <int D>
struct Raw {
  uint32_t codes[Layout<D>::kChunks][Layout<D>::kChunk / 8];
  uint32_t scales[Layout<D>::kChunks];
};

// `code_at`, `scale_at`: this lane's byte offsets from the first row.
template <int D>
__device__ __forceinline__ void load_rows(Raw<D>& r, const uint8_t* codes, const uint8_t* scales,
                                          uint32_t code_at, uint32_t scale_at) {
  using L = Layout<D>;
#pragma unroll
  for (int u = 0; u < L::kChunks; ++u) {
    typedef uint32_t Words __attribute__((ext_vector_type(L::kChunk / 8)));
    const Words w = *reinterpret_cast<const Words*>(codes + (code_at + u * 2 * L::kChunk));
#pragma unroll
    for (int j = 0; j < L::kChunk / 8; ++j) r.codes[u][j] = w[j];
    r.scales[u] = *reinterpret_cast<const uint32_t*>(scales + (scale_at + 4 * u));
  }
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

// Workgroups of a CU, by their registers and LDS.
constexpr int groups_per_cu(int dim, int tiles) {
  return dim == 64 ? (tiles == 1 ? 4 : 2) : dim == 128 ? (tiles == 1 ? 3 : 2) : 3 - tiles;
}

// kTiles tiles of 16 rows. kSplit: equal runs of all tiles; else workgroup (seq, head) alone.
template <int D, int kTiles, int kWaves, bool kSplit>
__global__ void __launch_bounds__(64 * kWaves, kSplit ? groups_per_cu(D, kTiles) * kWaves / 4 : kWaves / 4)
    attention_split_kernel(const AttentionArgs, int most, int most_blocks, int min_quota,
                           bool by_context, bool apart) {
  using L = Layout<D>;
  constexpr int kRows = 16 * kTiles;
  constexpr int kTileBytes = kTokens * L::kPitch;
  constexpr int kJoinPitch = D + 4;  // floats
  constexpr int kJoinBytes = 16 * kJoinPitch * 4;
  constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
  __shared__ __align__(16) char shared[kWaves * kWaveBytes];
  __shared__ float tops[kWaves][kRows], sums[kWaves][kRows];
  // The queries' operands stay in registers, or in LDS where those are taken.
  constexpr bool kQueriesInLds = D == 256 && kTiles == 2;
  constexpr int kSteps = L::kChunks * L::kSteps;
  __shared__ u32x4 queries[kQueriesInLds ? kTiles * kSteps * 64 : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane % 16, group4 = lane / 16;

  // Contexts that are few against the workgroups lie apart: each takes a whole number of equal runs,
  // so that no workgroup has two. Counted are at most 64 sequences then.
  const int begin = apart ? 0 : kBegin;
  Run run;
  Place place;
  if constexpr (kSplit) {
    const AttentionArgs& p = arguments();
    Counted counted = count_costs(p, most, kRows, begin, lane, 0);
    int64_t total = all_costs(p, most, kRows, begin, lane, counted);
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
    run.begin = blockIdx.x * run.quota;
    run.end = min(run.begin + run.quota, total);
    if (!by_context && threadIdx.x == 0) joints<D>(p)[blockIdx.x].parts = 0;
    if (run.begin >= total) return;
    place = find_place(p, most, kRows, begin, lane, run.begin, counted);
  } else {
    const AttentionArgs& p = arguments();
    place.block = blockIdx.x % most_blocks;
    place.head = blockIdx.x / most_blocks % p.cache.heads;
    place.seq = blockIdx.x / most_blocks / p.cache.heads;
    const Sequence s = sequence(p, place.seq);
    place.blocks = uniform(row_blocks(s, most, kRows));
    if (place.block >= place.blocks) return;
    place.at = 0;
    place.cost = uniform(block_tiles(s));
    run = {0, place.cost, place.cost};
  }
  // Where this lane's rows of 16 tokens start, and its place in the LDS tile.
  const uint32_t code_at = column * (D / 2) + group4 * (L::kChunk / 2);
  const uint32_t scale_byte = column * L::kScaleBytes + group4 * L::kChunk / kFp4Block;
  const uint32_t scale_at = scale_byte & ~3u, scale_turn = fp4_scale_turn(scale_byte % 4);
  char* const tile = shared + wave * kWaveBytes;
  char* const to = tile + column * L::kPitch + group4 * L::kChunk * 2;
  const char* const from = tile + (4 * group4 + column / 4) * L::kPitch + (column % 4) * 8;

  for (int64_t at = run.begin; at < run.end;) {
    const int seq = place.seq, kv_head = place.head;
    const AttentionArgs& p = arguments();
    const int page_mask = (1 << p.cache.page_shift) - 1;
    const Sequence s = sequence(p, seq);
    const int row0 = place.block * kRows, rows = min(s.rows - row0, kRows);
    const int take = int(min(int64_t(place.cost - place.at), run.end - at));
    // The run's share of the context's cost is its share of the tiles.
    const int tiles = block_tiles(s);
    const float share = float(tiles) / float(place.cost);
    auto tile_at = [&](int cost) {
      return s.first_tile(kTokens) +
             uniform(cost == place.cost ? tiles : min(int(float(cost) * share), tiles));
    };
    const int t_begin = tile_at(place.at), t_end = tile_at(place.at + take);

    // The lane's rows: their queries, and the tokens [low, high) that each attends to.
    int low[kTiles], high[kTiles];
    u32x4 q[kTiles][L::kChunks][L::kSteps];
    if (kQueriesInLds) __syncthreads();  // the last ones are read
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const int row = row0 + 16 * n + column;
      const bool live = row < s.rows;
      const int query = live ? row / p.group : 0;
      high[n] = live ? s.shift + query + 1 : 0;
      low[n] = p.window ? max(high[n] - p.window, 0) : 0;
      const uint16_t* src = p.q.data + int64_t(s.q_begin + query) * p.q.token_stride +
                            int64_t(kv_head * p.group + (live ? row % p.group : 0)) *
                                p.q.head_stride;
#pragma unroll
      for (int u = 0; u < L::kChunks; ++u)
#pragma unroll
        for (int j = 0; j < L::kSteps; ++j) {
          const int step = (n * L::kChunks + u) * L::kSteps + j;
          const u32x4* at =
              reinterpret_cast<const u32x4*>(src + (4 * u + group4) * L::kChunk + 8 * j);
          if constexpr (!kQueriesInLds)
            q[n][u][j] = *at ^ p.q_sign;
          else if (step % kWaves == wave)
            queries[step * 64 + lane] = *at ^ p.q_sign;
        }
      // Rows that are not there repeat a row that is; their results go nowhere.
    }
    if (kQueriesInLds) __syncthreads();

    f32x4 o[kTiles][D / 16];
    float reference[kTiles], sum[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[n][m] = f32x4{0, 0, 0, 0};
      reference[n] = kLowest;
      sum[n] = 0;
    }

    // This wave's tiles are t_begin + wave, + kWaves, ...; lane 2i + h holds where the page of half
    // h of the i-th begins, for 32 of them: in 16 bytes of codes and 8 of scales. Pages outside the
    // cache begin at 0 and have no bit in `in_cache`.
    struct {
      uint32_t k_codes, k_scales, v_codes, v_scales;
    } at_page;
    uint64_t in_cache = 0;
    auto load_pages = [&](int first) {
      const int t = first + (lane >> 1) * kWaves;
      const int token = t * kTokens + 16 * (lane & 1);
      int page = -1;
      if (t < t_end && token < s.context)
        page = p.page_table[int64_t(seq) * p.table_width + (token >> p.cache.page_shift)];
      const bool there = uint32_t(page) < uint32_t(p.cache.pages);
      in_cache = __ballot(there);
      const uint32_t safe = there ? page : 0;
      at_page = {safe * uint32_t(p.cache.k.code_stride >> 4),
                 safe * uint32_t(p.cache.k.scale_stride >> 3),
                 safe * uint32_t(p.cache.v.code_stride >> 4),
                 safe * uint32_t(p.cache.v.scale_stride >> 3)};
    };
    const int64_t head_row = int64_t(kv_head) << p.cache.page_shift;
    const uint8_t* const k_codes = p.cache.k.codes + head_row * (D / 2);
    const uint8_t* const v_codes = p.cache.v.codes + head_row * (D / 2);
    const uint8_t* const k_scales = p.cache.k.scales + head_row * L::kScaleBytes;
    const uint8_t* const v_scales = p.cache.v.scales + head_row * L::kScaleBytes;
    // Tile t, the i-th of those looked up.
    auto load = [&](Raw<D>(&raw)[2], const uint8_t* codes, uint32_t code_page,
                    const uint8_t* scales, uint32_t scale_page, int t, int i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t row = uint32_t(t * kTokens + 16 * h) & page_mask;
        const uint32_t code = __builtin_amdgcn_readlane(int(code_page), 2 * i + h);
        const uint32_t scale = __builtin_amdgcn_readlane(int(scale_page), 2 * i + h);
        load_rows<D>(raw[h], codes + (uint64_t(code) << 4), scales + (uint64_t(scale) << 3),
                     code_at + row * (D / 2), scale_at + row * L::kScaleBytes);
      }
    };

    // Keys and values of a tile each take the registers of the last as soon as those are used.
    // After the wave's last tile the loads go on with that one again: were they skipped, the waits
    // for those before would have to be for all.
    Raw<D> k[2], v[2];
    int t = t_begin + wave, i = 0, there = 3;
    if (t < t_end) {
      load_pages(t);
      load(k, k_codes, at_page.k_codes, k_scales, at_page.k_scales, t, 0);
      load(v, v_codes, at_page.v_codes, v_scales, at_page.v_scales, t, 0);
      there = int(in_cache & 3);
    }
    while (t < t_end) {
      const bool more = t + kWaves < t_end;
      const int t_next = more ? t + kWaves : t;
      if (more && ++i == 32) {
        load_pages(t_next);
        i = 0;
      }

      // Tiles that some row sees in part, or that are not whole.
      const bool edge = (t + 1) * kTokens > s.first_high || t * kTokens < s.last_low ||
                        there != 3;
      // Scores, lane: row `column`, tokens 4 * group4 + i of each half.
      f32x4 score[kTiles][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < kTiles; ++n) score[n][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < L::kChunks; ++u) {
#pragma unroll
        for (int j = 0; j < L::kSteps; ++j) {
          bf16x8 query[kTiles];
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
            query[n] = __builtin_bit_cast(
                bf16x8, kQueriesInLds ? queries[((n * L::kChunks + u) * L::kSteps + j) * 64 + lane]
                                      : q[n][u][j]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bf16x8 a = __builtin_bit_cast(
                bf16x8, fp4_to_bf16x8(k[h].codes[u][j], fp4_scale_in(k[h].scales[u], scale_turn)));
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
              score[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, query[n], score[n][h], 0, 0, 0);
          }
        }
      }
      load(k, k_codes, at_page.k_codes, k_scales, at_page.k_scales, t_next, i);

      uint32_t poisoned[2] = {0, 0};
      if (edge) {
        // Values of tokens past the context or of no page are zeros, and so are blocks that are
        // NaN, since some row may not see their token and its weight of 0 would not keep them out.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int token = t * kTokens + 16 * h + column;
          const bool real = (there >> h & 1) && token < s.context;
#pragma unroll
          for (int u = 0; u < L::kChunks; ++u) {
            if (!real || (v[h].scales[u] >> scale_byte % 4 * 8 & 0xFF) >= 253) {
              if (real) poisoned[h] |= 1u << ((4 * u + group4) * L::kChunk / kFp4Block);
#pragma unroll
              for (int j = 0; j < L::kSteps; ++j) v[h].codes[u][j] = 0;
              v[h].scales[u] = 0;
            }
          }
          poisoned[h] |= uint32_t(__shfl_xor(int(poisoned[h]), 16, 64));
          poisoned[h] |= uint32_t(__shfl_xor(int(poisoned[h]), 32, 64));
        }
      }
      wave_order();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < L::kChunks; ++u)
#pragma unroll
          for (int j = 0; j < L::kSteps; ++j)
            *reinterpret_cast<u32x4*>(to + 16 * h * L::kPitch + (4 * u * L::kChunk + 8 * j) * 2) =
                fp4_to_bf16x8(v[h].codes[u][j], fp4_scale_in(v[h].scales[u], scale_turn));
      wave_order();
      load(v, v_codes, at_page.v_codes, v_scales, at_page.v_scales, t_next, i);

      u32x4 weights[kTiles];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        float most = -__builtin_inff();
        if (edge) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int token = t * kTokens + 16 * h + 4 * group4 + j;
              const bool seen = (there >> h & 1) & (token >= low[n]) & (token < high[n]);
              score[n][h][j] = seen ? score[n][h][j] : -__builtin_inff();
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) most = fmaxf(most, score[n][h][j]);
        most *= p.scale_log2;
        if (__any(most > reference[n] + kSlack)) {
          most = fmaxf(most, __shfl_xor(most, 16, 64));
          most = fmaxf(most, __shfl_xor(most, 32, 64));
          most = fmaxf(most, reference[n]);
          const float factor = __builtin_amdgcn_exp2f(reference[n] - most);
          reference[n] = most;
          sum[n] *= factor;
#pragma unroll
          for (int m = 0; m < D / 16; ++m) o[n][m] *= factor;
        }
        float w[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[4 * h + j] =
                __builtin_amdgcn_exp2f(fmaf(score[n][h][j], p.scale_log2, -reference[n]));
            sum[n] += w[4 * h + j];
          }
        weights[n] = u32x4{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]),
                           pack_bf16x2(w[4], w[5]), pack_bf16x2(w[6], w[7])};
      }
#pragma unroll
      for (int m = 0; m < D / 16; ++m) {
        const u32x2 a = lds_read_transposed(from + 32 * m);
        const u32x2 b = lds_read_transposed(from + 16 * L::kPitch + 32 * m);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          o[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]}),
              __builtin_bit_cast(bf16x8, weights[n]), o[n][m], 0, 0, 0);
      }
      if (edge && __any(poisoned[0] | poisoned[1])) {
        for (int token = 0; token < kTokens; ++token) {
          const uint32_t blocks = uint32_t(__shfl(int(poisoned[token / 16]), token % 16, 64));
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
            if (t * kTokens + token >= low[n] && t * kTokens + token < high[n]) {
#pragma unroll
              for (int m = 0; m < D / 16; ++m)
                o[n][m] += blocks >> (m / 2) & 1 ? __builtin_nanf("") : 0.f;
            }
        }
      }
      there = int(in_cache >> (2 * i) & 3);
      t += kWaves;
    }

    // Joins the waves: one tile of rows at a time through LDS. Lane numbers are taken anew, so
    // that nothing of this is computed ahead and held through the loop above.
    {
    const AttentionArgs& p = arguments();
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, column = lane % 16, group4 = lane / 16;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      sum[n] += __shfl_xor(sum[n], 16, 64);
      sum[n] += __shfl_xor(sum[n], 32, 64);
      if (lane < 16) {
        tops[wave][16 * n + lane] = reference[n];
        sums[wave][16 * n + lane] = sum[n];
      }
    }
    __syncthreads();
    const bool whole = place.at == 0 && take == place.cost;
    const int part = 2 * blockIdx.x + (place.at == 0 ? 1 : 0);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float top = kLowest;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w][16 * n + column]);
      const float factor = __builtin_amdgcn_exp2f(reference[n] - top);
      float* join = reinterpret_cast<float*>(tile) + column * kJoinPitch + 4 * group4;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) *reinterpret_cast<f32x4*>(join + 16 * m) = o[n][m] * factor;
      __syncthreads();
      for (int i = thread; i < 16 * D / 4; i += 64 * kWaves) {
        const int r = i / (D / 4), row = 16 * n + r, channel = i % (D / 4) * 4;
        if (row >= rows) continue;
        float all = kLowest, l = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all = fmaxf(all, tops[w][row]);
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          l += sums[w][row] * __builtin_amdgcn_exp2f(tops[w][row] - all);
          x += *reinterpret_cast<const f32x4*>(shared + w * kWaveBytes +
                                               (r * kJoinPitch + channel) * 4);
        }
        if (!kSplit || whole) {
          write_row4(p, D, s.q_begin, row0 + row, kv_head, channel, x, all, l);
        } else {
          *reinterpret_cast<f32x4*>(part_sums<D, kTiles>(p, part) + row * D + channel) = x;
          if (channel == 0) {
            float* stats = part_stats<D, kTiles>(p, part) + row * 2;
            stats[0] = all;
            stats[1] = l;
          }
        }
      }
      __syncthreads();
    }
    if (kSplit && place.at == 0 && (by_context || !whole) && threadIdx.x == 0) {
      const int64_t last = at + place.cost - 1;
      joints<D>(p)[by_context ? (seq * p.cache.heads + kv_head) * most_blocks + place.block
                              : int(blockIdx.x)] = {
          whole ? 0 : int(last / run.quota) - int(blockIdx.x) + 1, int(blockIdx.x), s.q_begin,
          row0, rows, kv_head};
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
          place.blocks = uniform(row_blocks(next, most, kRows));
          place.cost = uniform(block_tiles(next)) + begin;
        } while (place.blocks == 0 && place.seq + 1 < p.seqs);
      }
    }
    }
  }
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

// Up to this many tiles of the longest context a workgroup takes a whole context: fewer where contexts
// leave most of the GPU idle. Whole and split, us: 16 contexts up to 2000 tokens of 8 heads of 128 14.3
// and 15.3, 64 of them 22.1 and 29.4, 4 13.5 and 12.1, one of 1100 9.6 and 11.8; 16 of 4 heads of 256
// 23.9 and 17.7. How long contexts are is known by the width of the page table alone here: a wide one of
// short contexts is split.
constexpr int whole_tiles(int dim, bool few) { return !few ? 64 : dim == 256 ? 32 : 48; }

template <int D, int kTiles>
hipError_t launch_split(const AttentionArgs& args, int most, hipStream_t stream) {
  const int64_t longest = (int64_t(args.table_width) << args.cache.page_shift) / kTokens;
  const int64_t span = args.window ? (int64_t(args.window) + args.max_q) / kTokens + 2 : longest;
  const int64_t rows = int64_t(args.max_q) * args.group;
  const int blocks = int(((rows < most ? rows : most) + 16 * kTiles - 1) / (16 * kTiles));
  const int64_t contexts = int64_t(args.seqs) * args.cache.heads * blocks;
  const int found = device_cu_count(), cus = found > 0 && found <= 256 ? found : 256;
  // Eight waves: 517 tokens of 8 key heads of 128 7.6 us, with four 8.3; 4 rows a sequence of 6
  // heads of 256, 64 contexts up to 1500, 25.5 and 32.4. Contexts past a launch's limit are split,
  // which takes any number.
  constexpr int kWholeWaves = 8;
  if ((longest < span ? longest : span) <= whole_tiles(D, 4 * contexts <= cus) &&
      launch_fits(contexts, 64 * kWholeWaves)) {
    attention_split_kernel<D, kTiles, kWholeWaves, false>
        <<<uint32_t(contexts), 64 * kWholeWaves, 0, stream>>>(args, most, blocks, 0, false, false);
    return hipGetLastError();
  }
  // Four waves a workgroup; with eight, in one workgroup a CU (two at 64 channels), us in turn: 32 contexts
  // up to 8000 tokens of 8 heads of 128 36.9 and 44.0, of 16 heads of 64 39.0 and 50.6; the longest would
  // gain, 64 up to 32768 264 and 258. Where the queries are in LDS eight waves share them: 16 x 4 rows up to 16000
  // of 4 heads of 256 51.4 us, with four 61.7. At D = 256 contexts that are few get one workgroup a CU and
  // so fewer parts to join: one of 131071 tokens of 4 heads 32.8 us, with two 34.8; 12 up to 9000 24.6 and
  // 25.6.
  constexpr int kWaves = D == 256 && kTiles == 2 ? 8 : 4;
  const int groups = D == 256 && contexts < 64 ? cus : cus * groups_per_cu(D, kTiles);
  static_assert(groups_per_cu(D, kTiles) <= 8 &&
                    2 * 256 * groups_per_cu(D, kTiles) * 16 * kTiles * 2 <=
                        kAttentionWorkspaceRows * 2 - 2048 * 8,
                "parts, statistics and descriptions fit the workspace");
  const bool by_context = contexts <= groups;
  // With more than three workgroups a context, us, and with runs of all: one of 100000 tokens of 4
  // heads of 256 28.1 and 31.5, 9 up to 90857 of 8 of 128 113 and 116, 4 up to 5000 14 and 17, 51 up
  // to 3006 of 4 (3.8 a context) 21.8 and 23.5; but 32 up to 8000 of 8 (3) 38.1 and 37.7, 16 x 5 rows
  // of 64 heads up to 16000 (2) 91 and 81.
  const bool apart = 3 * contexts < groups && args.seqs <= 64;
  attention_split_kernel<D, kTiles, kWaves, true>
      <<<groups, 64 * kWaves, 0, stream>>>(args, most, blocks, 2 * kWaves, by_context, apart);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  // More threads where a context has many parts. Whole calls with 1024 and with 256, us: one of 131071
  // tokens of 4 heads of 256, 64 parts each, 32.6 and 34.8; 32 up to 8000, 3 or 4 parts, 41.4 and 37.6.
  const bool many = groups > 16 * contexts;
  const auto join = many ? attention_join_kernel<D, kTiles, 1024> : attention_join_kernel<D, kTiles, 256>;
  join<<<dim3(by_context ? uint32_t(contexts) : groups, D / kJoinChannels), many ? 1024 : 256, 0,
         stream>>>(args, most, blocks, groups, by_context);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_split(const AttentionArgs& args, int dim, int most,
                                  hipStream_t stream) {
  if (most <= 16) {
    switch (dim) {
      case 64: return launch_split<64, 1>(args, most, stream);
      case 128: return launch_split<128, 1>(args, most, stream);
      default: return launch_split<256, 1>(args, most, stream);
    }
  }
  switch (dim) {
    case 64: return launch_split<64, 2>(args, most, stream);
    case 128: return launch_split<128, 2>(args, most, stream);
    default: return launch_split<256, 2>(args, most, stream);
  }
}

hipError_t launch_attention_fp4(const AttentionArgs& args, int dim, hipStream_t stream) {
  if (args.tokens == 0 || args.seqs == 0) return hipSuccess;
  const RowSplit rows = row_split(args.tokens, args.seqs, args.group, args.max_q);
  if (rows.split) {
    if (const hipError_t e = launch_attention_split(args, dim, rows.few, stream); e != hipSuccess)
      return e;
  }
  return rows.prompt ? launch_attention_prompt(args, dim, rows.few, stream) : hipSuccess;
}

}  // namespace ci8
