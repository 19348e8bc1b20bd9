// attention_fp4 (include/consumer_int8_attention.h): causal attention of BF16 queries over a
// paged cache of E2M1 values with power-of-two scales.
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp2(s_t - m),   s_t = q.k_t * scale * log2(e)
//
// in one pass with a running m. Rows are (token, query head of one key head) pairs, 16 a tile,
// so that the cache is read once for all heads that share it. A wave works alone on 32 tokens
// at a time:
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
// All statistics of a row sit in the lanes of its column. Waves of a workgroup take parts of
// the context and are joined in LDS.
#include "attention_launch.h"
#include "fp4_device.h"

namespace ci8 {
namespace {

constexpr int kRows = 16;    // query rows of a tile
constexpr int kTokens = 32;  // tokens a wave takes at once
constexpr float kLowest = -3.402823466e38f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Four values of one channel from four token rows, transposed on the way out of LDS: of each 16
// lanes, lanes 4j .. 4j+3 address row j (8 bytes each) and lane i gets column i of the rows.
__device__ __forceinline__ u32x2 lds_read_transposed(const char* p) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (lds_s16x4*)reinterpret_cast<const s16x4*>(p)));
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

// The codes and scales of 16 tokens' rows: this lane's token l % 16 and its chunks.
template <int D>
struct Raw {
  uint32_t codes[Layout<D>::kChunks][Layout<D>::kChunk / 8];
  uint32_t scales[Layout<D>::kChunks];
};

template <int D>
__device__ __forceinline__ Raw<D> load_rows(const uint8_t* codes, const uint8_t* scales, int lane,
                                            bool live) {
  using L = Layout<D>;
  Raw<D> r = {};
  if (!live) return r;
  const uint8_t* c = codes + (lane % 16) * (D / 2);
  const uint8_t* s = scales + (lane % 16) * L::kScaleBytes;
  const int group = lane / 16;
#pragma unroll
  for (int u = 0; u < L::kChunks; ++u) {
    const uint32_t* src =
        reinterpret_cast<const uint32_t*>(c + (4 * u + group) * (L::kChunk / 2));
#pragma unroll
    for (int w = 0; w < L::kChunk / 8; ++w) r.codes[u][w] = src[w];
    r.scales[u] = s[(4 * u + group) * L::kChunk / kFp4Block];
  }
  return r;
}

template <int D, int kWaves>
__global__ void __launch_bounds__(64 * kWaves) attention_kernel(const AttentionArgs p, int few) {
  using L = Layout<D>;
  constexpr int kTileBytes = kTokens * L::kPitch;
  constexpr int kJoinPitch = D + 4;  // floats
  constexpr int kJoinBytes = kRows * kJoinPitch * 4;
  constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
  __shared__ __align__(16) char shared[kWaves * kWaveBytes];
  __shared__ float top[kWaves][kRows], total[kWaves][kRows];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column = lane % 16, group4 = lane / 16;
  const int seq = blockIdx.y, kv_head = blockIdx.z;

  int q_begin = seq, q_count = 1;
  if (p.q_starts) {
    q_begin = min(max(p.q_starts[seq], 0), p.tokens);
    q_count = min(max(p.q_starts[seq + 1], q_begin), p.tokens) - q_begin;
  }
  const int row0 = blockIdx.x * kRows, rows = min(q_count, p.max_q) * p.group;
  if (row0 >= rows || rows <= few) return;
  const int page_size = 1 << p.cache.page_shift;
  const int64_t capacity = int64_t(p.table_width) << p.cache.page_shift;
  const int context = int(min(int64_t(max(p.context_lens[seq], 0)), capacity));

  // The lane's row: its query, and the tokens [low, high) that it attends to.
  const int row = row0 + column;
  const bool live_row = row < rows;
  const int query = live_row ? row / p.group : 0;
  const int head = kv_head * p.group + (live_row ? row % p.group : 0);
  const int high = live_row ? context - q_count + query + 1 : 0;
  const int low = p.window ? max(high - p.window, 0) : 0;
  // Tokens that any row of the tile attends to.
  const int last_query = min(row0 + kRows - 1, rows - 1) / p.group;
  const int tile_high = max(context - q_count + last_query + 1, 0);
  const int first_high = context - q_count + row0 / p.group + 1;
  const int tile_low = p.window ? max(first_high - p.window, 0) : 0;
  const int last_low = p.window ? max(tile_high - p.window, 0) : 0;

  u32x4 q[L::kChunks][L::kSteps];
#pragma unroll
  for (int u = 0; u < L::kChunks; ++u)
#pragma unroll
    for (int j = 0; j < L::kSteps; ++j) {
      q[u][j] = u32x4{0, 0, 0, 0};
      if (live_row)
        q[u][j] = *reinterpret_cast<const u32x4*>(
            p.q.data + int64_t(q_begin + query) * p.q.token_stride + head * p.q.head_stride +
            (4 * u + group4) * L::kChunk + 8 * j);
    }

  char* tile = shared + wave * kWaveBytes;
  f32x4 o[D / 16];
#pragma unroll
  for (int m = 0; m < D / 16; ++m) o[m] = f32x4{0, 0, 0, 0};
  float reference = kLowest, sum = 0;

  const int first_tile = tile_low / kTokens, tiles = (tile_high + kTokens - 1) / kTokens;
  for (int t = first_tile + wave; t < tiles; t += kWaves) {
    Raw<D> k[2], v[2];
    bool there[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int token = t * kTokens + 16 * h;
      int page = -1;
      if (token < context) page = p.page_table[int64_t(seq) * p.table_width +
                                               (token >> p.cache.page_shift)];
      there[h] = page >= 0 && page < p.cache.pages;
      const bool live = there[h] && token + lane % 16 < context;
      const int64_t row_in_page =
          (int64_t(kv_head) << p.cache.page_shift) + (token & (page_size - 1));
      const int64_t at = there[h] ? page : 0;
      k[h] = load_rows<D>(p.cache.k.codes + at * p.cache.k.code_stride + row_in_page * (D / 2),
                          p.cache.k.scales + at * p.cache.k.scale_stride +
                              row_in_page * L::kScaleBytes,
                          lane, live);
      v[h] = load_rows<D>(p.cache.v.codes + at * p.cache.v.code_stride + row_in_page * (D / 2),
                          p.cache.v.scales + at * p.cache.v.scale_stride +
                              row_in_page * L::kScaleBytes,
                          lane, live);
    }
    // Scores, lane: row `column`, tokens 4 * group4 + i of each half.
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < L::kChunks; ++u)
#pragma unroll
        for (int j = 0; j < L::kSteps; ++j)
          s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8,
                                 fp4_to_bf16x8(k[h].codes[u][j], fp4_scale(k[h].scales[u]))),
              __builtin_bit_cast(bf16x8, q[u][j]), s[h], 0, 0, 0);
    }
    // V into the LDS tile; rows that are not there hold zeros, and so do blocks that are NaN where
    // some row does not see their token: its weight of 0 would not keep them out.
    const bool edge = (t + 1) * kTokens > first_high || t * kTokens < last_low;
    uint32_t poisoned[2] = {0, 0};
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int u = 0; u < L::kChunks; ++u)
          if (v[h].scales[u] >= 253) {
            poisoned[h] |= 1u << ((4 * u + group4) * L::kChunk / kFp4Block);
#pragma unroll
            for (int j = 0; j < L::kSteps; ++j) v[h].codes[u][j] = 0;
            v[h].scales[u] = 0;
          }
        poisoned[h] |= uint32_t(__shfl_xor(int(poisoned[h]), 16, 64));
        poisoned[h] |= uint32_t(__shfl_xor(int(poisoned[h]), 32, 64));
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < L::kChunks; ++u)
#pragma unroll
        for (int j = 0; j < L::kSteps; ++j)
          *reinterpret_cast<u32x4*>(tile + (16 * h + lane % 16) * L::kPitch +
                                    ((4 * u + group4) * L::kChunk + 8 * j) * 2) =
              fp4_to_bf16x8(v[h].codes[u][j], fp4_scale(v[h].scales[u]));

    float most = kLowest;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = t * kTokens + 16 * h + 4 * group4 + i;
        const bool seen = there[h] && token >= low && token < high;
        s[h][i] = seen ? s[h][i] * p.scale_log2 : -__builtin_inff();
        most = fmaxf(most, s[h][i]);
      }
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64));
    if (__any(most > reference)) {
      const float next = fmaxf(most, reference);
      const float factor = __builtin_amdgcn_exp2f(reference - next);
      reference = next;
      sum *= factor;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[m] *= factor;
    }
    float w[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[4 * h + i] = __builtin_amdgcn_exp2f(s[h][i] - reference);
        sum += w[4 * h + i];
      }
    const u32x4 weights = {pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]),
                           pack_bf16x2(w[4], w[5]), pack_bf16x2(w[6], w[7])};
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const char* from = tile + (4 * group4 + column / 4) * L::kPitch + (column % 4) * 8;
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
      const u32x2 a = lds_read_transposed(from + 32 * m);
      const u32x2 b = lds_read_transposed(from + 16 * L::kPitch + 32 * m);
      o[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]}),
          __builtin_bit_cast(bf16x8, weights), o[m], 0, 0, 0);
    }
    if (edge && __any(poisoned[0] | poisoned[1])) {
      for (int i = 0; i < kTokens; ++i) {
        const uint32_t blocks = uint32_t(__shfl(int(poisoned[i / 16]), i % 16, 64));
        const int token = t * kTokens + i;
        if (token < low || token >= high) continue;
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
          if (blocks >> (m / 2) & 1) o[m] += __builtin_nanf("");
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (lane < kRows) {
    top[wave][lane] = reference;
    total[wave][lane] = sum;
  }
  __syncthreads();
  float highest = kLowest;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, top[w][column]);
  const float factor = __builtin_amdgcn_exp2f(reference - highest);
  float* join = reinterpret_cast<float*>(shared + wave * kWaveBytes);
#pragma unroll
  for (int m = 0; m < D / 16; ++m)
    *reinterpret_cast<f32x4*>(join + column * kJoinPitch + 16 * m + 4 * group4) = o[m] * factor;
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * D / 4; i += 64 * kWaves) {
    const int r = i / (D / 4), channel = i % (D / 4) * 4;
    if (row0 + r >= rows) continue;
    float m = kLowest, l = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, top[w][r]);
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      l += total[w][r] * __builtin_amdgcn_exp2f(top[w][r] - m);
      x += *reinterpret_cast<const f32x4*>(shared + w * kWaveBytes +
                                           (r * kJoinPitch + channel) * 4);
    }
    const float inv = l == 0 ? 0.f : 1.f / l;
    const int64_t at = int64_t(q_begin + (row0 + r) / p.group) * p.q.heads + kv_head * p.group +
                       (row0 + r) % p.group;
    u32x2 packed = {pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + at * D + channel) = packed;
    if (p.lse && channel == 0)
      p.lse[at] = l == 0 ? -__builtin_inff()
                         : (m + __builtin_log2f(l)) * 0.693147180559945309f;
  }
}

}  // namespace

hipError_t launch_attention_prompt(const AttentionArgs& args, int dim, int few, hipStream_t stream) {
  const int64_t rows = int64_t(args.max_q) * args.group;
  const dim3 grid(uint32_t((rows + kRows - 1) / kRows), args.seqs, args.cache.heads);
  switch (dim) {
    case 64: attention_kernel<64, 4><<<grid, 256, 0, stream>>>(args, few); break;
    case 128: attention_kernel<128, 4><<<grid, 256, 0, stream>>>(args, few); break;
    default: attention_kernel<256, 4><<<grid, 256, 0, stream>>>(args, few); break;
  }
  return hipGetLastError();
}

}  // namespace ci8
