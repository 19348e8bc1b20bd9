// token_probs and verify_drafts (include/consumer_int8_drafts.h).
//
//   p_i = exp2((l_i - m) c) / sum_j exp2((l_j - m) c),   c = log2(e) / temperature, m = max l
//
// (of halves of l and m above temperature 1: l_i - m itself may pass the finite numbers)
//
// and rejection sampling of drafted tokens against such rows. A vocabulary is one pass over memory
// and a few operations a value: bound by HBM for many rows, by launches and dependent loads for few.
// No sum depends on what finishes first: the same bits every time.
#include "ci8_device.h"
#include "sampling_launch.h"
#include "sampling_plan.h"

namespace ci8 {
namespace {

// Vectors that need not start on their size: a row starts wherever its stride puts it.
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
//
// A workgroup of 1024 threads a row holds the row in registers: it is read once, then its largest, the
// sum of its weights and the probabilities are computed from there (the exponential twice: weights
// in 32 bits would not fit beside). Where rows are few, several workgroups share one: each reads all
// of it, from the L2s, and writes a part; one launch, and nothing to wait for. Rows that are few and
// long take two kernels over their chunks instead (sampling_plan.h has both sides' times).
// Measured: 512 rows of 152000 BF16 logits 110 us, 4.2 TB/s of the 5.1 that a copy reaches; 1000 of 50001
// in FP32 89, 4.5; one of 32000 5.8, 3 of it the launch. Plain stores: nontemporal ones 163.

// Registers hold 163840 BF16 or 81920 FP32 values of a row, or 32768 in less code, which a launch of
// few workgroups has to fetch first: one row of 32000 5.4 us, with room for 163840 10.8.
constexpr int kFewHeld = 8;
constexpr int kPackValues = 4, kRowStep = kRowThreads * kPackValues;  // values that all threads take
static_assert(kRowStep == kProbsPart && kFewVocab <= (kFewHeld + 1) * kRowStep);

// Four values of a row as they lie there: neighbouring lanes load and store what lies side by side.
template <bool kBf16>
struct Pack {
  static constexpr int kBytes = kBf16 ? 2 : 4;  // of a value
  uint32_t raw[kBytes];
  __device__ __forceinline__ void load(const void* row, int at) {
    typedef uint32_t __attribute__((ext_vector_type(kBytes), aligned(2))) Loose;
    const Loose x =
        *reinterpret_cast<const Loose*>(static_cast<const char*>(row) + int64_t(at) * kBytes);
#pragma unroll
    for (int j = 0; j < kBytes; ++j) raw[j] = x[j];
  }
  // Past the end -inf.
  __device__ __forceinline__ void load(const void* row, int at, int vocab) {
    if (at + 4 <= vocab) return load(row, at);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kBf16) {
        const uint32_t x = at + j < vocab ? static_cast<const uint16_t*>(row)[at + j] : 0xFF80u;
        raw[j / 2] = j % 2 ? raw[j / 2] | x << 16 : x;
      } else {
        raw[j] = at + j < vocab ? static_cast<const uint32_t*>(row)[at + j] : 0xFF800000u;
      }
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (!kBf16)
      return __uint_as_float(raw[j]);
    else
      return j % 2 ? bf16_hi(raw[j / 2]) : bf16_lo(raw[j / 2]);
  }
};
__device__ __forceinline__ void store4(float* row, int at, int vocab, const float (&x)[4]) {
  if (at + 4 <= vocab) {
    *reinterpret_cast<loose_f32x4*>(row + at) = loose_f32x4{x[0], x[1], x[2], x[3]};
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + j < vocab) row[at + j] = x[j];
}

// The weight of a logit against `top`, exp2((l - top) c) with c = log2(e) / temperature. Above temperature 1
// the difference is one of halves (exact, but for logits below 2^-125) and c twice as large: whole, it may
// pass the finite numbers where the exponent is small. At 1 or below such a difference has a weight of 0
// either way. 512 x 152000 BF16 logits 111 us, by the whole difference 110.
// c is held among the finite numbers above 0, which leave 0 * c at 0 and -inf * c at -inf; NaN for
// temperatures that are none.
struct Weigh {
  float part, c;
  __device__ __forceinline__ explicit Weigh(float temperature) {
    part = temperature > 1 ? 0.5f : 1.f;
    const float inverse = (temperature > 1 ? 2.8853900817779268f : 1.4426950408889634f) / temperature;
    c = temperature >= 0 ? fminf(fmaxf(inverse, __uint_as_float(1)), 3.402823466e38f)
                         : __builtin_nanf("");
  }
  __device__ __forceinline__ float operator()(float logit, float top) const {
    return __builtin_amdgcn_exp2f(fmaf(logit, part, -top * part) * c);
  }
};

// Workgroup (token, part of `length` values). A thread holds kHeld packs, and one more that may pass the
// end or be of any further step; others between are loaded for each use.
template <bool kBf16, int kHeld>
__global__ void __launch_bounds__(kRowThreads) probs_kernel(const ProbsArgs p, int length, int parts) {
  __shared__ float room[kRowThreads / 64];
  const int token = blockIdx.x / parts, part = blockIdx.x % parts;
  const void* const row =
      static_cast<const char*>(p.logits) + token * p.logit_stride * (kBf16 ? 2 : 4);
  float* const out = p.probs + token * p.prob_stride;
  const float temperature = p.temperature ? p.temperature[token] : 1.f;
  const int vocab = p.vocab, mine = kPackValues * int(threadIdx.x);
  const int whole = vocab / kRowStep;  // steps that do not pass the end
  Pack<kBf16> held[kHeld], last;
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (i < whole) held[i].load(row, mine + i * kRowStep);
  last.load(row, mine + whole * kRowStep, vocab);
  // f(values, place) of all packs of the thread.
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < whole) f(held[i], mine + i * kRowStep);
    for (int i = kHeld; i < whole; ++i) {
      Pack<kBf16> x;
      x.load(row, mine + i * kRowStep);
      f(x, mine + i * kRowStep);
    }
    f(last, mine + whole * kRowStep);
  };
  float top = -kInf;
  each([&](const Pack<kBf16>& x, int) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, x[j]);
  });
  top = reduce_all<kRowThreads>(top, room, larger);
  const int begin = part * length, end = min(begin + length, vocab);
  if (temperature == 0) {
    // 1 at the first of the largest; NaN if any logit is, nothing where none is above -inf.
    int first = 0x7FFFFFFF;
    each([&](const Pack<kBf16>& x, int at) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (x[j] == top && top > -kInf) first = min(first, at + j);  // past the end is -inf
        if (x[j] != x[j]) first = -1;
      }
    });
    first = reduce_all<kRowThreads>(first, reinterpret_cast<int*>(room), smaller);
    for (int at = begin + mine; at < end; at += kRowStep) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = first < 0 ? __builtin_nanf("") : at + j == first ? 1.f : 0.f;
      store4(out, at, vocab, y);
    }
    return;
  }
  // Where nothing is above -inf all weights are 0. +inf gives NaN, as inf - inf is.
  const Weigh weight(temperature);
  const float against = top == -kInf ? 0.f : top;
  float sums[2] = {0, 0};
  each([&](const Pack<kBf16>& x, int) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[j % 2] += weight(x[j], against);
  });
  const float sum = reduce_all<kRowThreads>(sums[0] + sums[1], room, add<float>);
  const float scale = sum == 0 ? 0.f : 1.f / sum;
  each([&](const Pack<kBf16>& x, int at) __attribute__((always_inline)) {
    if (at - mine < begin || at - mine >= end) return;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = weight(x[j], against) * scale;
    store4(out, at, vocab, y);
  });
}

// What a chunk of a row adds up to: its largest logit, and the sum of the weights against it (against
// 0 where nothing is above -inf, so that all are 0); at temperature 0 the place of the first that is
// largest: negative if a logit is NaN, past all places if nothing is above -inf.
struct RowPart {
  float top, sum;
};
__device__ __forceinline__ float against(float top) { return top == -kInf ? 0.f : top; }

// Workgroup (token, chunk). A thread has kChunkPacks packs of it at most.
template <bool kBf16>
struct ChunkOfRow {
  int token, begin, end;
  const void* row;
  float temperature;
  Pack<kBf16> held[kChunkPacks];
  __device__ __forceinline__ ChunkOfRow(const ProbsArgs& p, int length, int chunks) {
    token = blockIdx.x / chunks;
    begin = int(blockIdx.x % chunks) * length;
    end = min(begin + length, p.vocab);
    row = static_cast<const char*>(p.logits) + token * p.logit_stride * (kBf16 ? 2 : 4);
    temperature = p.temperature ? p.temperature[token] : 1.f;
    begin += kPackValues * int(threadIdx.x);
#pragma unroll
    for (int i = 0; i < kChunkPacks; ++i) held[i].load(row, at(i), end);
  }
  __device__ __forceinline__ int at(int i) const { return begin + i * kSampleThreads * kPackValues; }
};

template <bool kBf16>
__global__ void __launch_bounds__(kSampleThreads)
    probs_parts_kernel(const ProbsArgs p, int length, int chunks) {
  __shared__ float room[kSampleThreads / 64];
  const ChunkOfRow<kBf16> chunk(p, length, chunks);
  float top = -kInf;
#pragma unroll
  for (int i = 0; i < kChunkPacks; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, chunk.held[i][j]);
  RowPart part;
  part.top = top = reduce_all<kSampleThreads>(top, room, larger);
  if (chunk.temperature == 0) {
    int first = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < kChunkPacks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = chunk.held[i][j];
        if (x == top && top > -kInf) first = min(first, chunk.at(i) + j);
        if (x != x) first = -1;
      }
    part.sum = __int_as_float(
        reduce_all<kSampleThreads>(first, reinterpret_cast<int*>(room), smaller));
  } else {
    const Weigh weight(chunk.temperature);
    float sums[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kChunkPacks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[j % 2] += weight(chunk.held[i][j], against(top));
    part.sum = reduce_all<kSampleThreads>(sums[0] + sums[1], room, add<float>);
  }
  if (threadIdx.x == 0) reinterpret_cast<RowPart*>(p.workspace)[blockIdx.x] = part;
}

// Joins the chunks' parts in each of them, and writes it.
template <bool kBf16>
__global__ void __launch_bounds__(kSampleThreads)
    probs_write_kernel(const ProbsArgs p, int length, int chunks) {
  __shared__ float room[kSampleThreads / 64];
  const ChunkOfRow<kBf16> chunk(p, length, chunks);
  const RowPart* parts = reinterpret_cast<const RowPart*>(p.workspace) + int64_t(chunk.token) * chunks;
  RowPart mine = {-kInf, 0.f};  // chunks are no more than threads
  if (int(threadIdx.x) < chunks) mine = parts[threadIdx.x];
  const float top = reduce_all<kSampleThreads>(mine.top, room, larger);
  float* const out = p.probs + chunk.token * p.prob_stride;
  float y[4];
  if (chunk.temperature == 0) {
    const int place = __float_as_int(mine.sum);
    int first = 0x7FFFFFFF;
    if (int(threadIdx.x) < chunks && (place < 0 || mine.top == top)) first = place;
    first = reduce_all<kSampleThreads>(first, reinterpret_cast<int*>(room), smaller);
#pragma unroll
    for (int i = 0; i < kChunkPacks; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        y[j] = first < 0 ? __builtin_nanf("") : chunk.at(i) + j == first ? 1.f : 0.f;
      store4(out, chunk.at(i), chunk.end, y);
    }
    return;
  }
  const Weigh weight(chunk.temperature);
  float sum = mine.sum;
  if (sum != 0) sum *= weight(mine.top, against(top));
  sum = reduce_all<kSampleThreads>(sum, room, add<float>);
  const float scale = sum == 0 ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < kChunkPacks; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = weight(chunk.held[i][j], against(top)) * scale;
    store4(out, chunk.at(i), chunk.end, y);
  }
}

// ---- verify_drafts ----------------------------------------------------------------------
//
// Which drafts stand takes one value of p and q a row, all loaded at once, a row a lane; a vocabulary is
// read where none stands any more, and between the children of a drafter's row. Weights, sums and
// comparisons are in 64 bits: a running sum over 150000 values in 32 would lose tokens of less than 6e-8
// of it.
//
// Chains and certain choices need sums at the end alone: every wave follows its sequence and adds up a
// chunk of what is left, then a second kernel finds the chunk and the token. 64 chains of 9 over 152000
// tokens 22.4 us: the sums 16.5 (78 MB, 4.7 TB/s), the token 8.3, a chain of dependent loads.
//
// Trees of a drafter's tokens need a sum for every child but the last that fails. Several workgroups
// share a sequence: all follow it, each sums its chunk, and sums go from one to the others through the
// workspace, which a first kernel fills with what is no sum. A workgroup that waits in vain (another may
// not run yet) adds up the missing chunks itself, so every wait ends, and to the same result. 16 trees
// of 32 rows over 128000 tokens take as long as the one that asks for most sums before its last: 25 us with
// two of them, 31 to 35 with four, 43 with six, so 4 a sum; with one workgroup a sequence 62.7.

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
  int row;
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

// Tokens of rejected rows in [begin, end) to `skip`; how many.
__device__ __forceinline__ int skipped(uint64_t rejected, int token, int lane, int begin, int end,
                                       int* skip) {
  const bool mine = has_lane(rejected, lane) && token >= begin && token < end;
  const uint64_t all = __ballot(mine);
  if (mine) skip[lanes_before(all)] = token;
  return __builtin_popcountll(all);
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
                                          int* places) {
  const double sum = scan_all<kThreads>(mine, room);
  const int past = sum > bar && mine > 0 ? int(threadIdx.x) : 0x7FFFFFFF;
  int found = reduce_all<kThreads>(past, places, smaller);
  if (found == 0x7FFFFFFF) {
    const int last = mine > 0 ? -int(threadIdx.x) : 1;
    found = reduce_all<kThreads>(last, places, smaller);
    found = found > 0 ? -1 : -found;
  }
  __syncthreads();
  if (int(threadIdx.x) == found) room[0] = sum - mine;
  __syncthreads();
  before = found < 0 ? 0 : room[0];
  return found;
}

// One wave: what is known of the sequence before any vocabulary is read.
__device__ __forceinline__ void write_path(const VerifyArgs& p, const Rows& rows, int seq, int lane,
                                           int path, int accepted) {
  for (int i = lane; i < rows.count; i += 64) p.path[rows.begin + i] = i == lane ? path : -1;
  if (lane == 0) p.accepted[seq] = rows.count ? accepted : 0;
}

constexpr uint64_t kNoSum = ~uint64_t(0);  // a NaN, which no sum is

__global__ void __launch_bounds__(kClearThreads) verify_clear_kernel(uint64_t* sums, int count) {
  const int i = blockIdx.x * kClearThreads + threadIdx.x;
  if (i < count) sums[i] = kNoSum;
}

// A chunk of a sequence's vocabulary, and the sums of all its chunks.
template <int kThreads>
struct Cluster {
  int seq, chunk, chunks, length, vocab;
  uint64_t* shared_sums;  // of this sequence
  double* room;           // LDS, a value a wave
  double* sums;           // LDS, a value a chunk: the last sums
  int* missing;           // LDS
  int round;

  __device__ __forceinline__ int begin(int i) const { return i * length; }
  __device__ __forceinline__ int end(int i) const { return min(i * length + length, vocab); }

  // The sum of weights over the vocabulary. weights_in(begin, end) gives those of a chunk.
  template <typename F>
  __device__ __forceinline__ double total(F weights_in) {
    const double own = sum_weights<kThreads>(weights_in(begin(chunk), end(chunk)), begin(chunk),
                                             end(chunk), room);
    if (chunks == 1) {
      if (threadIdx.x == 0) sums[0] = own;
      __syncthreads();
      return own;
    }
    uint64_t* const slots = shared_sums + round * chunks;
    ++round;
    if (threadIdx.x == 0) {
      __hip_atomic_store(slots + chunk, __builtin_bit_cast(uint64_t, own), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      *missing = 0;
    }
    __syncthreads();
    if (int(threadIdx.x) < chunks) {
      uint64_t bits = kNoSum;
      for (int i = 0; i < kMostPolls && bits == kNoSum; ++i) {
        bits = __hip_atomic_load(slots + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (bits == kNoSum) __builtin_amdgcn_s_sleep(1);
      }
      sums[threadIdx.x] = __builtin_bit_cast(double, bits);
      if (bits == kNoSum) *missing = 1;
    }
    __syncthreads();
    if (*missing) {
      for (int i = 0; i < chunks; ++i) {
        if (__builtin_bit_cast(uint64_t, sums[i]) != kNoSum) continue;
        const double sum = sum_weights<kThreads>(weights_in(begin(i), end(i)), begin(i), end(i), room);
        __syncthreads();
        if (threadIdx.x == 0) sums[i] = sum;
        __syncthreads();
      }
    }
    double mine = 0;
    if (int(threadIdx.x) < chunks) mine = sums[threadIdx.x];
    return reduce_all<kThreads>(mine, room, add<double>);
  }
};

// A sequence, as far as its drafts stand. Lane l has row l: its parent, its token and, in the lane's
// values, what the parent's rows have for it.
struct Followed {
  Stop stop;
  double number;       // of row 0
  int token;           // of the lane's row
  int path, accepted;  // path: in lane i the i-th accepted row
};
// Every wave of every workgroup that needs it follows the sequence, and all come to the same.
// left_after(stop, token): what is left of a drafter's row at a stop; only trees of its tokens ask.
template <typename F>
__device__ __forceinline__ Followed follow(const VerifyArgs& p, const Rows& rows, int lane,
                                           F left_after) {
  const int count = min(rows.count, kMostRows), row = rows.begin + lane;
  int parent = -1;
  float pt = 0, qt = 0, u = 0;
  Followed x = {{0.0, 0, 0}, 0.0, -1, lane == 0 ? 0 : -1, 1};
  if (lane < count) {
    u = fminf(fmaxf(p.uniforms[row], 0.f), kMostUniform);
    if (lane > 0) {
      parent = p.parents ? p.parents[row] : lane - 1;
      if (parent >= lane) parent = -1;
      x.token = token_of(p, row);
    }
    if (parent >= 0 && x.token >= 0) {
      pt = clean(p.target[(rows.begin + parent) * p.target_stride + x.token]);
      if (p.draft) qt = clean(p.draft[(rows.begin + parent) * p.draft_stride + x.token]);
    }
  }
  x.number = at_lane(double(u), 0);
  double left = 1;
  uint64_t children = __ballot(parent == 0);
  while (children) {
    const int i = __builtin_ctzll(children);
    children &= children - 1;
    const double number = at_lane(double(u), i), q = at_lane(double(qt), i);
    double w = at_lane(double(pt), i);
    bool stands;
    if (p.draft) {
      w = fmax(w - x.stop.taken * q, 0.0);
      stands = number * (left * q) < w;
    } else {
      const int id = __builtin_amdgcn_readlane(x.token, i);
      if (__ballot(has_lane(x.stop.rejected, lane) && x.token == id)) w = 0;
      stands = number * left < w;
    }
    if (stands) {
      if (lane == x.accepted) x.path = i;
      ++x.accepted;
      x.stop = {0.0, 0, i};
      left = 1;
      children = __ballot(parent == i);
    } else if (p.draft) {
      x.stop.taken += left;
      if (children) left = left_after(x.stop, x.token);
    } else {
      left -= w;
      x.stop.rejected |= uint64_t(1) << i;
    }
  }
  return x;
}

// Weights at a stop in [begin, end); skip: room of the wave for tokens that have none.
__device__ __forceinline__ Weights weights_at(const VerifyArgs& p, const Rows& rows, const Stop& stop,
                                              int token, int lane, int begin, int end, int* skip) {
  const int64_t at = rows.begin + stop.row;
  const int skips = skipped(stop.rejected, token, lane, begin, end, skip);
  return {p.target + at * p.target_stride, stop.taken > 0 ? p.draft + at * p.draft_stride : nullptr,
          stop.taken, skip, skips};
}

// Writes the first token of [begin, end) whose running sum of weights passes `level`, or the last that
// has a weight; -1 if none has. One workgroup alone writes a sequence's: stores of two would meet in
// different L2s.
template <int kThreads>
__device__ __forceinline__ void pick(const Weights& weights, int begin, int end, double level,
                                     double* room, int* places, int64_t* next) {
  const int each = ((end - begin + kThreads - 1) / kThreads + 3) / 4 * 4;
  const int first = min(begin + each * int(threadIdx.x), end), last = min(first + each, end);
  double part = 0, w[4];
  for (int at = first; at < last; at += 4) {
    weights.load(at, last, w);
    part += (w[0] + w[1]) + (w[2] + w[3]);
  }
  double sum;
  const int found = first_past<kThreads>(part, level, sum, room, places);
  int token = -1;
  if (int(threadIdx.x) != max(found, 0)) return;
  bool past = found < 0;
  for (int at = first; at < last && !past; at += 4) {
    weights.load(at, last, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum += w[j];
      if (!past && w[j] > 0) {
        token = at + j;
        past = sum > level;
      }
    }
  }
  *next = token;
}

// Workgroup (sequence, chunk), where sums may be needed on the way, or a workgroup has it all.
template <int kThreads>
__global__ void __launch_bounds__(kThreads)
    verify_cluster_kernel(const VerifyArgs p, int length, int chunks, int rounds) {
  constexpr int kWaves = kThreads / 64;
  __shared__ double room[kWaves], sums[kMostChunks];
  __shared__ int places[kWaves], missing, skip[kWaves][kMostRows];
  const int seq = blockIdx.x / chunks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Cluster<kThreads> cluster = {seq, int(blockIdx.x % chunks), chunks, length, p.vocab,
                               static_cast<uint64_t*>(p.workspace) + int64_t(seq) * rounds * chunks,
                               room, sums, &missing, 0};
  const Rows rows = rows_of(p, seq);
  auto total = [&](const Stop& stop, int token) {
    return cluster.total([&](int begin, int end) {
      return weights_at(p, rows, stop, token, lane, begin, end, skip[wave]);
    });
  };
  Followed x = follow(p, rows, lane, total);
  if (cluster.chunk == 0 && wave == 0) write_path(p, rows, seq, lane, x.path, x.accepted);
  auto none = [&]() {
    if (cluster.chunk == 0 && threadIdx.x == 0) p.next[seq] = -1;
  };
  if (rows.count == 0) return none();

  // The chunk that the first row's number falls in, then the token. Where no weight is left, the
  // target's own.
  double all = total(x.stop, x.token);
  if (all == 0 && (x.stop.taken > 0 || x.stop.rejected)) {
    x.stop.taken = 0;
    x.stop.rejected = 0;
    all = total(x.stop, x.token);
  }
  if (all == 0) return none();
  const double bar = x.number * all;
  double before = 0;
  if (chunks > 1) {
    const double mine = int(threadIdx.x) < chunks ? sums[threadIdx.x] : 0;
    if (first_past<kThreads>(mine, bar, before, room, places) != cluster.chunk) return;
  }
  const int begin = cluster.begin(cluster.chunk), end = cluster.end(cluster.chunk);
  const Weights weights = weights_at(p, rows, x.stop, x.token, lane, begin, end, skip[wave]);
  pick<kThreads>(weights, begin, end, bar - before, room, places, p.next + seq);
}

// Chains, and certain choices: sums are needed at the end alone, so a second kernel joins them. A wave
// adds up a chunk; the workspace has a sum for each, then the stops.
__device__ __forceinline__ Stop* stops(const VerifyArgs& p, int chunks) {
  return reinterpret_cast<Stop*>(static_cast<double*>(p.workspace) + int64_t(p.seqs) * chunks);
}
__global__ void __launch_bounds__(kSampleThreads)
    verify_sums_kernel(const VerifyArgs p, int length, int chunks) {
  __shared__ int skip[kSampleThreads / 64][kMostRows];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, index = blockIdx.x * (kSampleThreads / 64) + wave;
  const int seq = index / chunks, chunk = index % chunks;
  if (seq >= p.seqs) return;
  const Rows rows = rows_of(p, seq);
  const Followed x = follow(p, rows, lane, [](const Stop&, int) { return 0.0; });
  if (chunk == 0) {
    write_path(p, rows, seq, lane, x.path, x.accepted);
    if (lane == 0) stops(p, chunks)[seq] = x.stop;
  }
  if (rows.count == 0) return;
  const int begin = chunk * length, end = min(begin + length, p.vocab);
  const Weights weights = weights_at(p, rows, x.stop, x.token, lane, begin, end, skip[wave]);
  double sum = 0, w[4];
#pragma unroll 4
  for (int at = begin + 4 * lane; at < end; at += 256) {
    weights.load(at, end, w);
    sum += (w[0] + w[1]) + (w[2] + w[3]);
  }
#pragma unroll
  for (int step = 32; step >= 1; step /= 2) sum += __shfl_xor(sum, step, 64);
  if (lane == 0) static_cast<double*>(p.workspace)[index] = sum;
}

// A workgroup a sequence.
__global__ void __launch_bounds__(kPickThreads)
    verify_pick_kernel(const VerifyArgs p, int length, int chunks) {
  constexpr int kThreads = kPickThreads, kWaves = kThreads / 64;
  __shared__ double room[kWaves];
  __shared__ int places[kWaves], skip[kWaves][kMostRows];
  const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows rows = rows_of(p, seq);
  if (rows.count == 0) {
    if (threadIdx.x == 0) p.next[seq] = -1;
    return;
  }
  const double mine = int(threadIdx.x) < chunks
                          ? static_cast<const double*>(p.workspace)[int64_t(seq) * chunks + threadIdx.x]
                          : 0;
  Stop stop = stops(p, chunks)[seq];
  const double number = fminf(fmaxf(p.uniforms[rows.begin], 0.f), kMostUniform);
  int token = -1;
  if (has_lane(stop.rejected, lane)) token = token_of(p, rows.begin + lane);
  const double all = reduce_all<kThreads>(mine, room, add<double>);
  double bar = number * all, before;
  const int chunk = first_past<kThreads>(mine, bar, before, room, places);
  int begin = chunk * length, end = min(begin + length, p.vocab);
  if (chunk < 0) {
    // Where no weight is left, the target's own.
    begin = 0;
    end = p.vocab;
    stop.taken = 0;
    stop.rejected = 0;
    const Weights weights = weights_at(p, rows, stop, token, lane, begin, end, skip[wave]);
    bar = number * sum_weights<kThreads>(weights, begin, end, room);
    before = 0;
  }
  const Weights weights = weights_at(p, rows, stop, token, lane, begin, end, skip[wave]);
  pick<kThreads>(weights, begin, end, bar - before, room, places, p.next + seq);
}

}  // namespace

hipError_t launch_token_probs(const ProbsArgs& args, bool bf16, hipStream_t stream) {
  if (args.tokens == 0) return hipSuccess;
  const Chunks c = probs_chunks(args.tokens, args.vocab);
  const uint32_t tokens = uint32_t(args.tokens);
  if (probs_in_chunks(args.tokens, args.vocab, c, bf16)) {
    const auto parts = bf16 ? probs_parts_kernel<true> : probs_parts_kernel<false>;
    parts<<<tokens * c.count, kSampleThreads, 0, stream>>>(args, c.length, c.count);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const auto write = bf16 ? probs_write_kernel<true> : probs_write_kernel<false>;
    write<<<tokens * c.count, kSampleThreads, 0, stream>>>(args, c.length, c.count);
    return hipGetLastError();
  }
  // In place a row has one workgroup, which has read a value before it writes there.
  const bool in_place = args.logits == args.probs;
  const Chunks parts = in_place ? Chunks{args.vocab, 1} : probs_parts(args.tokens, args.vocab);
  const bool few = args.vocab < kFewVocab;
  const auto kernel = bf16 ? (few ? probs_kernel<true, kFewHeld> : probs_kernel<true, 40>)
                           : (few ? probs_kernel<false, kFewHeld> : probs_kernel<false, 20>);
  kernel<<<tokens * parts.count, kRowThreads, 0, stream>>>(args, parts.length, parts.count);
  return hipGetLastError();
}

hipError_t launch_verify_drafts(const VerifyArgs& args, hipStream_t stream) {
  if (args.seqs == 0) return hipSuccess;
  const Chunks c = verify_chunks(args.seqs, args.vocab, args.draft && args.parents);
  const uint32_t workgroups = uint32_t(args.seqs) * c.count;
  if (c.count == 1) {
    verify_cluster_kernel<kRowThreads>
        <<<workgroups, kRowThreads, 0, stream>>>(args, c.length, 1, kMostRounds);
    return hipGetLastError();
  }
  if (args.draft && args.parents) {
    const int sums = args.seqs * c.count * kMostRounds;
    verify_clear_kernel<<<(sums + kClearThreads - 1) / kClearThreads, kClearThreads, 0, stream>>>(
        static_cast<uint64_t*>(args.workspace), sums);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    verify_cluster_kernel<kSampleThreads>
        <<<workgroups, kSampleThreads, 0, stream>>>(args, c.length, c.count, kMostRounds);
    return hipGetLastError();
  }
  constexpr int kWaves = kSampleThreads / 64;
  verify_sums_kernel<<<(workgroups + kWaves - 1) / kWaves, kSampleThreads, 0, stream>>>(args, c.length,
                                                                                       c.count);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  verify_pick_kernel<<<uint32_t(args.seqs), kPickThreads, 0, stream>>>(args, c.length, c.count);
  return hipGetLastError();
}

}  // namespace ci8
