// token_probs and verify_drafts (include/consumer_int8_drafts.h).
//
//   p_i = exp2((l_i - m) c) / sum_j exp2((l_j - m) c),   c = log2(e) / temperature, m = max l
//
// and rejection sampling of drafted tokens against such rows. A vocabulary is one or two passes over
// memory and a few operations a value: bound by HBM for many rows, by launches and dependent loads for
// few, so a row is cut into chunks that fill the GPU, whose sums are joined by a second kernel in a
// fixed order (no atomics, the same bits every time).
//
// Which drafts stand takes one value of p and q a row, all loaded at once, a row a lane. Only where none
// stands any more is a vocabulary read. Weights, sums and comparisons are in 64 bits: a running sum over
// 150000 values in 32 would lose tokens of less than 6e-8 of it.
#include "ci8_device.h"
#include "sampling_launch.h"
#include "sampling_plan.h"

namespace ci8 {
namespace {

// Vectors that need not start on their size: a row starts wherever its stride puts it.
typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) loose_u32x4;
typedef float __attribute__((ext_vector_type(4), aligned(4))) loose_f32x4;

constexpr float kInf = __builtin_inff();

// Sums, and largest, over a workgroup of kThreads; every thread gets the result. `room`: a value a
// wave, free again after the next barrier but one.
template <int kThreads, typename T, typename Op>
__device__ __forceinline__ T reduce_all(T v, T* room, Op op) {
#pragma unroll
  for (int step = 32; step >= 1; step /= 2) v = op(v, __shfl_xor(v, step, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
  __syncthreads();
  T all = room[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) all = op(all, room[w]);
  return all;
}
template <typename T>
__device__ __forceinline__ T add(T a, T b) { return a + b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ int smaller(int a, int b) { return min(a, b); }

// ---- token_probs ------------------------------------------------------------------------

// Eight values of a row from `at` on; past the end -inf.
template <bool kBf16>
__device__ __forceinline__ void load8(const void* row, int at, int vocab, float (&x)[8]) {
  if (at + 8 <= vocab) {
    if constexpr (kBf16) {
      const loose_u32x4 raw =
          *reinterpret_cast<const loose_u32x4*>(static_cast<const uint16_t*>(row) + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = bf16_lo(raw[j]);
        x[2 * j + 1] = bf16_hi(raw[j]);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const loose_f32x4 raw =
            *reinterpret_cast<const loose_f32x4*>(static_cast<const float*>(row) + at + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * h + j] = raw[j];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = -kInf;
    if (at + j < vocab)
      x[j] = kBf16 ? bf16_to_f32(static_cast<const uint16_t*>(row)[at + j])
                   : static_cast<const float*>(row)[at + j];
  }
}
__device__ __forceinline__ void store8(float* row, int at, int vocab, const float (&x)[8]) {
  if (at + 8 <= vocab) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<loose_f32x4*>(row + at + 4 * h) =
          loose_f32x4{x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at + j < vocab) row[at + j] = x[j];
}

// c = log2(e) / temperature, held among the finite numbers above 0, which leave 0 * c at 0 and
// -inf * c at -inf; NaN for temperatures that are none.
__device__ __forceinline__ float inverse_of(float temperature) {
  const float c = 1.4426950408889634f / temperature;
  return temperature >= 0 ? fminf(fmaxf(c, __uint_as_float(1)), 3.402823466e38f)
                          : __builtin_nanf("");
}

// What a part of a row adds up to: its largest logit, and the sum of the weights against it (against
// 0 where nothing is above -inf, so that all are 0); at temperature 0 the place of the first that is
// largest (negative if a logit is NaN, past all places if nothing is above -inf).
struct RowPart {
  float top, sum;
};
__device__ __forceinline__ float against(float top) { return top == -kInf ? 0.f : top; }
// Weights of 8 logits against `top`, c as above. +inf is NaN, as inf - inf is.
__device__ __forceinline__ float weigh8(float (&x)[8], float top, float c) {
  float s[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = __builtin_amdgcn_exp2f((x[j] - top) * c);
    s[j % 2] += x[j];
  }
  return s[0] + s[1];
}

template <bool kBf16, int kThreads>
__device__ __forceinline__ RowPart row_part(const void* row, int begin, int end, float temperature,
                                            float* room) {
  RowPart part;
  float top = -kInf;
  bool nan = false;
  float x[8];
  for (int at = begin + 8 * int(threadIdx.x); at < end; at += 8 * kThreads) {
    load8<kBf16>(row, at, end, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top = fmaxf(top, x[j]);
      nan = nan || x[j] != x[j];
    }
  }
  top = reduce_all<kThreads>(top, room, larger);
  part.top = top;
  if (temperature == 0) {
    int first = 0x7FFFFFFF;
    for (int at = begin + 8 * int(threadIdx.x); at < end; at += 8 * kThreads) {
      load8<kBf16>(row, at, end, x);
#pragma unroll
      for (int j = 7; j >= 0; --j)
        if (x[j] == top && top > -kInf) first = min(first, at + j);
    }
    first = reduce_all<kThreads>(nan ? -1 : first, reinterpret_cast<int*>(room), smaller);
    part.sum = __int_as_float(first);
    return part;
  }
  const float c = inverse_of(temperature);
  float sum = 0;
  for (int at = begin + 8 * int(threadIdx.x); at < end; at += 8 * kThreads) {
    load8<kBf16>(row, at, end, x);
    sum += weigh8(x, against(top), c);
  }
  part.sum = reduce_all<kThreads>(sum, room, add<float>);
  return part;
}

// Writes [begin, end) of a row: of weights against `top`, whose sum over the row is `sum`; at
// temperature 0 1 at `first`.
template <bool kBf16, int kThreads>
__device__ __forceinline__ void write_part(const ProbsArgs& p, const void* row, int token, int begin,
                                           int end, float temperature, const RowPart& all) {
  float* const out = p.probs + token * p.prob_stride;
  const bool greedy = temperature == 0;
  const int first = __float_as_int(all.sum);
  const float c = inverse_of(temperature);
  // Where nothing is above -inf, all weights are 0 and so is their sum.
  const float scale = greedy ? 0.f : all.sum == 0 ? 0.f : 1.f / all.sum;
  float x[8];
  for (int at = begin + 8 * int(threadIdx.x); at < end; at += 8 * kThreads) {
    load8<kBf16>(row, at, end, x);
    if (greedy) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = first < 0 ? __builtin_nanf("") : at + j == first ? 1.f : 0.f;
    } else {
      weigh8(x, against(all.top), c);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= scale;
    }
    store8(out, at, end, x);
  }
}

template <bool kBf16>
__device__ __forceinline__ const void* logit_row(const ProbsArgs& p, int token) {
  return static_cast<const char*>(p.logits) + token * p.logit_stride * (kBf16 ? 2 : 4);
}
__device__ __forceinline__ float temperature_of(const ProbsArgs& p, int token) {
  return p.temperature ? p.temperature[token] : 1.f;
}

// Workgroup (token, chunk): the chunk's part goes to the workspace.
template <bool kBf16>
__global__ void __launch_bounds__(kSampleThreads)
    probs_parts_kernel(const ProbsArgs p, int length, int chunks) {
  __shared__ float room[kSampleThreads / 64];
  const int token = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int begin = chunk * length, end = min(begin + length, p.vocab);
  const RowPart part = row_part<kBf16, kSampleThreads>(logit_row<kBf16>(p, token), begin, end,
                                                       temperature_of(p, token), room);
  if (threadIdx.x == 0) reinterpret_cast<RowPart*>(p.workspace)[blockIdx.x] = part;
}

// Joins the parts of the row and writes the chunk.
template <bool kBf16>
__global__ void __launch_bounds__(kSampleThreads)
    probs_write_kernel(const ProbsArgs p, int length, int chunks) {
  __shared__ float room[kSampleThreads / 64];
  const int token = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int begin = chunk * length, end = min(begin + length, p.vocab);
  const float temperature = temperature_of(p, token);
  const RowPart* parts = reinterpret_cast<const RowPart*>(p.workspace) + int64_t(token) * chunks;
  RowPart all;
  float top = -kInf;
  for (int i = threadIdx.x; i < chunks; i += kSampleThreads) top = fmaxf(top, parts[i].top);
  all.top = top = reduce_all<kSampleThreads>(top, room, larger);
  if (temperature == 0) {
    int first = 0x7FFFFFFF;
    for (int i = threadIdx.x; i < chunks; i += kSampleThreads) {
      const int at = __float_as_int(parts[i].sum);
      if (at < 0 || parts[i].top == top) first = min(first, at);
    }
    all.sum = __int_as_float(
        reduce_all<kSampleThreads>(first, reinterpret_cast<int*>(room), smaller));
  } else {
    const float c = inverse_of(temperature);
    float sum = 0;
    for (int i = threadIdx.x; i < chunks; i += kSampleThreads)
      if (parts[i].sum != 0)
        sum += parts[i].sum * __builtin_amdgcn_exp2f((parts[i].top - against(top)) * c);
    all.sum = reduce_all<kSampleThreads>(sum, room, add<float>);
  }
  write_part<kBf16, kSampleThreads>(p, logit_row<kBf16>(p, token), token, begin, end, temperature, all);
}

// A workgroup a row.
template <bool kBf16>
__global__ void __launch_bounds__(kRowThreads) probs_rows_kernel(const ProbsArgs p) {
  __shared__ float room[kRowThreads / 64];
  const int token = blockIdx.x;
  const void* const row = logit_row<kBf16>(p, token);
  const float temperature = temperature_of(p, token);
  const RowPart all = row_part<kBf16, kRowThreads>(row, 0, p.vocab, temperature, room);
  write_part<kBf16, kRowThreads>(p, row, token, 0, p.vocab, temperature, all);
}

// ---- verify_drafts ----------------------------------------------------------------------

constexpr float kMostUniform = 1 - 0x1p-24f;  // the largest number below 1

__device__ __forceinline__ float clean(float x) { return x > 0 && x < kInf ? x : 0.f; }

// A row's token, -1 if it is none.
__device__ __forceinline__ int token_of(const VerifyArgs& p, int row) {
  const int64_t id = p.ids[row];
  return id >= 0 && id < p.vocab ? int(id) : -1;
}

// Where a sequence's way ends: the row, and what of its weights is gone.
struct Stop {
  double taken;       // times the drafter's row
  uint64_t rejected;  // rows whose tokens have none
  int row, pad;
};
constexpr int kMostRows = 64;

struct Rows {
  int begin, count;
};
__device__ __forceinline__ Rows rows_of(const VerifyArgs& p, int seq) {
  const int begin = min(max(p.q_starts[seq], 0), p.tokens);
  return {begin, min(max(p.q_starts[seq + 1], begin), p.tokens) - begin};
}

// Weights of four tokens from `at` on at a stop, 0 past `end`. skip: those tokens have none.
struct Weights {
  const float* target;
  const float* draft;  // null: nothing of it is taken
  double taken;
  const int* skip;
  int skips;
  __device__ __forceinline__ void load(int at, int end, double (&w)[4]) const {
    float t[4], d[4] = {0, 0, 0, 0};
    if (at + 4 <= end) {
      const loose_f32x4 x = *reinterpret_cast<const loose_f32x4*>(target + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = x[j];
      if (draft) {
        const loose_f32x4 y = *reinterpret_cast<const loose_f32x4*>(draft + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = y[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[j] = at + j < end ? target[at + j] : 0.f;
        if (draft) d[j] = at + j < end ? draft[at + j] : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = fmax(double(clean(t[j])) - taken * double(clean(d[j])), 0.0);
    for (int i = 0; i < skips; ++i) {
      const int j = skip[i] - at;
      if (uint32_t(j) < 4) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (n == j) w[n] = 0;
      }
    }
  }
};

template <int kThreads>
__device__ __forceinline__ double sum_weights(const Weights& weights, int begin, int end,
                                              double* room) {
  double sum = 0, w[4];
  for (int at = begin + 4 * int(threadIdx.x); at < end; at += 4 * kThreads) {
    weights.load(at, end, w);
    sum += (w[0] + w[1]) + (w[2] + w[3]);
  }
  return reduce_all<kThreads>(sum, room, add<double>);
}

__device__ __forceinline__ double at_lane(double v, int lane) {
  const int64_t bits = __builtin_bit_cast(int64_t, v);
  const uint32_t low = __builtin_amdgcn_readlane(int(bits), lane);
  const uint32_t high = __builtin_amdgcn_readlane(int(bits >> 32), lane);
  return __builtin_bit_cast(double, int64_t(uint64_t(high) << 32 | low));
}

// Follows sequence rows.begin .. as far as its drafts stand. Every wave does so, and all come to the
// same. kSums: a row may have several children of a drafter's row, so sums over it are needed.
// path: in lane i the i-th accepted row.
template <int kThreads, bool kSums>
__device__ __forceinline__ Stop follow(const VerifyArgs& p, const Rows& rows, int lane, int& path,
                                       int& accepted, int& token, double* room) {
  const int count = min(rows.count, kMostRows), row = rows.begin + lane;
  int parent = -1;
  float pt = 0, qt = 0, u = 0;
  token = -1;
  if (lane < count) {
    u = fminf(fmaxf(p.uniforms[row], 0.f), kMostUniform);
    if (lane > 0) {
      parent = p.parents ? p.parents[row] : lane - 1;
      if (parent >= lane) parent = -1;
      token = token_of(p, row);
    }
    if (parent >= 0 && token >= 0) {
      pt = clean(p.target[(rows.begin + parent) * p.target_stride + token]);
      if (p.draft) qt = clean(p.draft[(rows.begin + parent) * p.draft_stride + token]);
    }
  }
  Stop stop = {0.0, 0, 0, 0};
  double left = 1;
  path = lane == 0 ? 0 : -1;
  accepted = 1;
  uint64_t children = __ballot(parent == 0);
  while (children) {
    const int i = __builtin_ctzll(children);
    children &= children - 1;
    const double number = at_lane(double(u), i), q = at_lane(double(qt), i);
    double w = at_lane(double(pt), i);
    bool stands;
    if (p.draft) {
      w = fmax(w - stop.taken * q, 0.0);
      stands = number * (left * q) < w;
    } else {
      const int id = __builtin_amdgcn_readlane(token, i);
      if (__ballot((stop.rejected >> lane & 1) && token == id)) w = 0;
      stands = number * left < w;
    }
    if (stands) {
      if (lane == accepted) path = i;
      ++accepted;
      stop = {0.0, 0, i, 0};
      left = 1;
      children = __ballot(parent == i);
    } else if (p.draft) {
      stop.taken += left;
      if (kSums && children) {
        const int64_t at = rows.begin + stop.row;
        const Weights weights = {p.target + at * p.target_stride, p.draft + at * p.draft_stride,
                                 stop.taken, nullptr, 0};
        left = sum_weights<kThreads>(weights, 0, p.vocab, room);
      }
    } else {
      left -= w;
      stop.rejected |= uint64_t(1) << i;
    }
  }
  return stop;
}

// One wave: what is known of the sequence before any vocabulary is read.
__device__ __forceinline__ void write_path(const VerifyArgs& p, const Rows& rows, int seq, int lane,
                                           int path, int accepted) {
  for (int i = lane; i < rows.count; i += 64) p.path[rows.begin + i] = i == lane ? path : -1;
  if (lane == 0) p.accepted[seq] = rows.count ? accepted : 0;
}

// The workspace: a sum for each chunk of each sequence, then the stops.
__device__ __forceinline__ double* chunk_sums(const VerifyArgs& p) {
  return static_cast<double*>(p.workspace);
}
__device__ __forceinline__ Stop* stops(const VerifyArgs& p, int chunks) {
  return reinterpret_cast<Stop*>(chunk_sums(p) + int64_t(p.seqs) * chunks);
}

// Trees of a drafter's tokens: a workgroup a sequence follows it.
__global__ void __launch_bounds__(kRowThreads) verify_follow_kernel(const VerifyArgs p, int chunks) {
  __shared__ double room[kRowThreads / 64];
  const int seq = blockIdx.x, lane = threadIdx.x & 63;
  const Rows rows = rows_of(p, seq);
  int path, accepted, token;
  const Stop stop = follow<kRowThreads, true>(p, rows, lane, path, accepted, token, room);
  if (threadIdx.x < 64) write_path(p, rows, seq, lane, path, accepted);
  if (threadIdx.x == 0) stops(p, chunks)[seq] = stop;
}

// Tokens of rejected rows in [begin, end) to `skip`; how many.
__device__ __forceinline__ int skipped(uint64_t rejected, int token, int lane, int begin, int end,
                                       int* skip) {
  const bool mine = (rejected >> lane & 1) && token >= begin && token < end;
  const uint64_t all = __ballot(mine);
  if (mine) skip[__builtin_popcountll(all & ((uint64_t(1) << lane) - 1))] = token;
  return __builtin_popcountll(all);
}

__device__ __forceinline__ Weights weights_at(const VerifyArgs& p, const Rows& rows, const Stop& stop,
                                              const int* skip, int skips) {
  const int64_t at = rows.begin + stop.row;
  return {p.target + at * p.target_stride, stop.taken > 0 ? p.draft + at * p.draft_stride : nullptr,
          stop.taken, skip, skips};
}

// Workgroup (sequence, chunk): the sum of the chunk's weights where the sequence stops. kFollowed: that
// is known.
template <bool kFollowed>
__global__ void __launch_bounds__(kSampleThreads)
    verify_sums_kernel(const VerifyArgs p, int length, int chunks) {
  __shared__ double room[kSampleThreads / 64];
  __shared__ int skip[kSampleThreads / 64][kMostRows];
  const int seq = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x & 63;
  const Rows rows = rows_of(p, seq);
  Stop stop;
  int token = -1;
  if (kFollowed) {
    stop = stops(p, chunks)[seq];
  } else {
    int path, accepted;
    stop = follow<kSampleThreads, false>(p, rows, lane, path, accepted, token, room);
    if (chunk == 0 && threadIdx.x < 64) write_path(p, rows, seq, lane, path, accepted);
    if (chunk == 0 && threadIdx.x == 0) stops(p, chunks)[seq] = stop;
  }
  if (rows.count == 0) return;
  const int begin = chunk * length, end = min(begin + length, p.vocab), wave = threadIdx.x >> 6;
  const int skips = skipped(stop.rejected, token, lane, begin, end, skip[wave]);
  const double sum =
      sum_weights<kSampleThreads>(weights_at(p, rows, stop, skip[wave], skips), begin, end, room);
  if (threadIdx.x == 0) chunk_sums(p)[blockIdx.x] = sum;
}

// Inclusive sums over the workgroup's threads.
template <int kThreads>
__device__ __forceinline__ double scan_all(double v, double* room) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const double other = __shfl_up(v, step, 64);
    if (lane >= step) v += other;
  }
  __syncthreads();
  if (lane == 63) room[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += room[w];
  return v;
}

// The first thread whose running sum passes `bar`; if rounding leaves none, the last that adds
// anything; -1 if none does. before: the sum in front of it.
template <int kThreads>
__device__ __forceinline__ int first_past(double mine, double bar, double& before, double* room,
                                          int* places, bool share) {
  const double sum = scan_all<kThreads>(mine, room);
  const double total = share ? bar * reduce_all<kThreads>(mine, room, add<double>) : bar;
  const int past = sum > total && mine > 0 ? int(threadIdx.x) : 0x7FFFFFFF;
  int found = reduce_all<kThreads>(past, places, smaller);
  if (found == 0x7FFFFFFF) {
    const int last = mine > 0 ? -int(threadIdx.x) : 1;
    found = reduce_all<kThreads>(last, places, smaller);
    found = found > 0 ? -1 : -found;
  }
  __syncthreads();
  if (int(threadIdx.x) == found) room[0] = sum - mine, room[1] = total;
  __syncthreads();
  before = found < 0 ? 0 : room[0];
  return found;
}

// The first token of [begin, end) whose running sum of weights passes `bar` (share: `bar` times their
// sum); -1 where no token has a weight.
template <int kThreads>
__device__ __forceinline__ int pick(const Weights& weights, int begin, int end, double bar, bool share,
                                    double* room, int* places) {
  const int each = ((end - begin + kThreads - 1) / kThreads + 3) / 4 * 4;
  const int first = min(begin + each * int(threadIdx.x), end), last = min(first + each, end);
  double mine = 0, w[4];
  for (int at = first; at < last; at += 4) {
    weights.load(at, last, w);
    mine += (w[0] + w[1]) + (w[2] + w[3]);
  }
  double before;
  const int found = first_past<kThreads>(mine, bar, before, room, places, share);
  if (found < 0) return -1;
  const double level = room[1];
  if (int(threadIdx.x) == found) {
    int token = -1;
    bool past = false;
    for (int at = first; at < last && !past; at += 4) {
      weights.load(at, last, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        before += w[j];
        if (!past && w[j] > 0) {
          token = at + j;
          past = before > level;
        }
      }
    }
    places[0] = token;
  }
  __syncthreads();
  return places[0];
}

// A workgroup a sequence: the chunk that the number falls in, then the token.
__global__ void __launch_bounds__(kRowThreads)
    verify_pick_kernel(const VerifyArgs p, int length, int chunks) {
  constexpr int kThreads = kRowThreads;
  __shared__ double room[kThreads / 64];
  __shared__ int places[kThreads / 64];
  __shared__ int skip[kThreads / 64][kMostRows];
  const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows rows = rows_of(p, seq);
  if (rows.count == 0) {
    if (threadIdx.x == 0) p.next[seq] = -1;
    return;
  }
  const Stop stop = stops(p, chunks)[seq];
  const double u = fminf(fmaxf(p.uniforms[rows.begin], 0.f), kMostUniform);
  const double mine = int(threadIdx.x) < chunks ? chunk_sums(p)[int64_t(seq) * chunks + threadIdx.x] : 0;
  double before;
  const int chunk = first_past<kThreads>(mine, u, before, room, places, true);
  int token;
  if (chunk >= 0) {
    const double bar = room[1] - before;
    int id = -1;
    if (stop.rejected >> lane & 1) id = token_of(p, rows.begin + lane);
    const int begin = chunk * length, end = min(begin + length, p.vocab);
    const int skips = skipped(stop.rejected, id, lane, begin, end, skip[wave]);
    __syncthreads();
    token = pick<kThreads>(weights_at(p, rows, stop, skip[wave], skips), begin, end, bar, false, room,
                           places);
  } else {
    const Weights all = {p.target + (rows.begin + stop.row) * p.target_stride, nullptr, 0.0, nullptr, 0};
    token = pick<kThreads>(all, 0, p.vocab, u, true, room, places);
  }
  if (threadIdx.x == 0) p.next[seq] = token;
}

}  // namespace

hipError_t launch_token_probs(const ProbsArgs& args, bool bf16, hipStream_t stream) {
  if (args.tokens == 0) return hipSuccess;
  if (args.tokens >= kManyRows) {
    const auto kernel = bf16 ? probs_rows_kernel<true> : probs_rows_kernel<false>;
    kernel<<<uint32_t(args.tokens), kRowThreads, 0, stream>>>(args);
    return hipGetLastError();
  }
  const Chunks c = vocab_chunks(args.tokens, args.vocab);
  const uint32_t grid = uint32_t(args.tokens) * c.count;
  const auto parts = bf16 ? probs_parts_kernel<true> : probs_parts_kernel<false>;
  parts<<<grid, kSampleThreads, 0, stream>>>(args, c.length, c.count);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const auto write = bf16 ? probs_write_kernel<true> : probs_write_kernel<false>;
  write<<<grid, kSampleThreads, 0, stream>>>(args, c.length, c.count);
  return hipGetLastError();
}

hipError_t launch_verify_drafts(const VerifyArgs& args, hipStream_t stream) {
  if (args.seqs == 0) return hipSuccess;
  const Chunks c = vocab_chunks(args.seqs, args.vocab);
  const bool followed = args.draft && args.parents;
  if (followed) {
    verify_follow_kernel<<<uint32_t(args.seqs), kRowThreads, 0, stream>>>(args, c.count);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  const auto sums = followed ? verify_sums_kernel<true> : verify_sums_kernel<false>;
  sums<<<uint32_t(args.seqs) * c.count, kSampleThreads, 0, stream>>>(args, c.length, c.count);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  verify_pick_kernel<<<uint32_t(args.seqs), kRowThreads, 0, stream>>>(args, c.length, c.count);
  return hipGetLastError();
}

}  // namespace ci8
