// qk_norm_rope, append_fp4 and unpack_fp4 (include/consumer_int8_attention.h): what stands
// between a layer's projected tokens and its attention.
//
//   y = rotate(x * (1 / sqrt(mean(x^2) + eps)) * w)     for each query and key head,
//
// rounded to BF16, or for appended keys (and values as they are) to E2M1 codes with a
// power-of-two scale for 32 channels. Every operation is rounded once in a stated order (no
// contraction, squares summed in a tree of neighbours), so that codes are reproducible.
//
// About two operations a byte: bound by HBM, and by latency for a few tokens. A lane holds 8
// channels (16 bytes) of a head, so a head is 8, 16 or 32 lanes and a wave covers 8, 4 or 2
// heads at once; sums, maxima and the rotation's partners are DPP exchanges inside those lanes
// (through LDS they took as long as the memory) and nothing needs LDS memory. A wave keeps one
// token's angles for all its heads. Measured, with bytes read and written, calls in a HIP
// graph: 4096 tokens of 24 + 4 heads of 256 24.1 us, 4.9 TB/s, 9261 of 16 + 16 of 64 with three axes 20.3
// us, 3.9 TB/s, where a large copy reaches 5.0; one token of 32 + 8 heads of 128 2.9 us. Three axes that
// turn all 128 channels are far from that, 2617 tokens of 40 + 8 heads 49 us and with one axis 15.3: the
// angles of several axes are loaded one channel at a time.
#include "attention_launch.h"
#include "attention_plan.h"
#include "fp4_device.h"

#pragma clang fp contract(off)

namespace ci8 {
namespace {

__device__ __forceinline__ void unpack8(const u32x4& raw, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(raw[j]);
    x[2 * j + 1] = bf16_hi(raw[j]);
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
               pack_bf16x2(x[6], x[7])};
}

// A value from another lane by a DPP control: 0xB1 and 0x4E are lane ^ 1 and lane ^ 2, 0x141 and
// 0x140 reverse 8 and 16 lanes, which is lane ^ 4 and lane ^ 8 of values that 4 and 8 share.
template <int kControl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, 0xF, 0xF, true));
}
template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kControl, 0xF, 0xF, true));
}

// Sums of neighbours, of pairs of those and so on, over kLanes lanes (8, 16 or 32).
template <int kLanes>
__device__ __forceinline__ float tree_sum(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  if constexpr (kLanes > 8) v += dpp<0x140>(v);
  if constexpr (kLanes > 16) {
    // Both rows of 16 lanes of each 32, in either operand.
    const auto rows =
        __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(rows[0]) + __int_as_float(rows[1]);
  }
  return v;
}

// Largest |x| of a block of 32 channels (4 lanes), as FP32 bits: a NaN is larger than all.
__device__ __forceinline__ uint32_t block_amax(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  m = max(m, dpp<0xB1>(m));
  return max(m, dpp<0x4E>(m));
}

// Cosine and signed sine of this lane's 8 channels: y = x cos + partner sin.
struct Angles {
  float cos[8], sin[8];
};

template <int D>
__device__ __forceinline__ Angles load_angles(const RotationView& r, int64_t at, int64_t tokens,
                                              int token, int channel) {
  Angles a;
  const int half = r.rot / 2;
  const bool second = !r.interleaved && channel >= half;
  const int first = r.interleaved ? channel / 2 : second ? channel - half : channel;
  // One axis for all pairs: four channels a load. (Reading axis_of here as well took every call 0.4 to
  // 0.8 us, with it or without: 1024 tokens of 32 + 8 heads of 128 8.2 us and 7.6.)
  if (r.axes == 1 && !r.axis_of) {
    const bool inside = at >= 0 && at < r.rows;
    const float* row = r.table + (inside ? at : 0) * r.rot + first;
    if (r.interleaved) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(row);
      const f32x4 s = *reinterpret_cast<const f32x4*>(row + half);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a.cos[j] = c[j / 2];
        a.sin[j] = j % 2 ? s[j / 2] : -s[j / 2];
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(row + 4 * h);
        const f32x4 s = *reinterpret_cast<const f32x4*>(row + half + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a.cos[4 * h + j] = c[j];
          a.sin[4 * h + j] = second ? s[j] : -s[j];
        }
      }
    }
    if (!inside) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a.cos[j] = __builtin_nanf("");
    }
    return a;
  }
  // Rows of the table for up to four axes, the same in all lanes; -1 outside it.
  constexpr int kAxes = 4;
  int64_t rows[kAxes];
#pragma unroll
  for (int i = 0; i < kAxes; ++i) {
    rows[i] = i < r.axes ? r.positions[i * tokens + token] : -1;
    if (rows[i] >= r.rows) rows[i] = -1;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int pair = first + (r.interleaved ? j / 2 : j);
    const int axis = r.axis_of[pair];
    int64_t row = -1;
    if (r.axes <= kAxes) {
#pragma unroll
      for (int i = 0; i < kAxes; ++i) row = axis == i ? rows[i] : row;
    } else if (axis >= 0 && axis < r.axes) {
      row = r.positions[axis * tokens + token];
      if (row >= r.rows) row = -1;
    }
    const float* values = r.table + (row < 0 ? 0 : row) * r.rot + pair;
    const float s = values[half];
    a.cos[j] = row < 0 ? __builtin_nanf("") : values[0];
    a.sin[j] = (r.interleaved ? j % 2 : int(second)) ? s : -s;
  }
  return a;
}

// x <- x / rms(x) * weight over the D / 8 lanes of a head.
template <int D>
__device__ __forceinline__ void norm8(float (&x)[8], const float* weight, float eps) {
  float s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = x[2 * j] * x[2 * j] + x[2 * j + 1] * x[2 * j + 1];
  const float sum = tree_sum<D / 8>((s[0] + s[1]) + (s[2] + s[3]));
  const float inv = 1.f / __builtin_sqrtf(sum * (1.f / D) + eps);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(weight + 4 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * h + j] = x[4 * h + j] * inv * w[j];
  }
}

// The values of lane ^ step, for a step that is a power of two: without LDS. Others by lane number.
__device__ __forceinline__ void exchange8(const float (&x)[8], float (&other)[8], int step, int lane,
                                          int from) {
  switch (step) {
    case 1:
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = dpp<0xB1>(x[j]);
      break;
    case 2:
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = dpp<0x4E>(x[j]);
      break;
    case 4:  // 8 lanes reversed (lane ^ 7), then 4 (lane ^ 3)
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = dpp<0x1B>(dpp<0x141>(x[j]));
      break;
    case 8:  // a row of 16 turned by 8
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = dpp<0x128>(x[j]);
      break;
    case 16:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_int(x[j]),
                                                           __float_as_int(x[j]), false, false);
        other[j] = __int_as_float(lane & 16 ? rows[0] : rows[1]);
      }
      break;
    default:
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = __shfl(x[j], from, 64);
  }
}

template <int D>
__device__ __forceinline__ void rotate8(float (&x)[8], const Angles& a, const RotationView& r,
                                        int lane, int channel) {
  float other[8];
  if (r.interleaved) {
#pragma unroll
    for (int j = 0; j < 8; ++j) other[j] = x[j ^ 1];
  } else {
    // The pair's other half: rot / 16 lanes on or back. Lanes past rot get anything.
    const int step = r.rot / 16;
    const int from = channel < r.rot / 2 ? lane + step : channel < r.rot ? lane - step : lane;
    exchange8(x, other, step, lane, from);
  }
  if (channel < r.rot) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * a.cos[j] + other[j] * a.sin[j];
  }
}

// Eight channels of a row into the cache.
template <int D>
__device__ __forceinline__ void store_fp4(const float (&x)[8], const Fp4Rows& rows, int64_t page,
                                          int row_in_page, int channel, bool live) {
  const uint32_t byte = fp4_scale_byte(block_amax(x));
  const uint32_t codes = fp4_codes8(x, byte);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(rows.codes + page * rows.code_stride +
                               int64_t(row_in_page) * (D / 2) + channel / 2) = codes;
  if (channel % kFp4Block == 0)
    rows.scales[page * rows.scale_stride + int64_t(row_in_page) * (D / kFp4Block) +
                channel / kFp4Block] = uint8_t(byte);
}

// A wave takes kGroups groups of 512 / D heads of one token; a group is of queries, of keys or
// of values alone. All loads of the wave come first.
template <int D, bool kAppend, int kGroups>
__global__ void __launch_bounds__(kNormThreads)
    norm_rope_kernel(const NormRopeArgs p, int q_groups, int k_groups, int groups, int chunks) {
  constexpr int kLanes = D / 8, kHeads = 64 / kLanes;
  const int lane = threadIdx.x & 63, channel = lane % kLanes * 8;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int token = wave / chunks, first = wave % chunks * kGroups;
  if (token >= p.tokens) return;
  // The token's position and slot come first: its angles' and rows' places wait for them.
  const int64_t position = p.rotation.rot ? p.rotation.positions[token] : 0;
  int64_t slot = -1;
  if constexpr (kAppend) slot = p.slots[token];

  u32x4 raw[kGroups];
  int head[kGroups];
  bool live[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int group = first + i;
    const bool is_q = group < q_groups, is_k = !is_q && group < q_groups + k_groups;
    const HeadsView& in = is_q ? p.q : is_k ? p.k : p.v;
    head[i] = (is_q ? group : is_k ? group - q_groups : group - q_groups - k_groups) * kHeads +
              lane / kLanes;
    live[i] = group < groups && head[i] < in.heads;
    raw[i] = u32x4{0, 0, 0, 0};
    if (live[i])
      raw[i] = *reinterpret_cast<const u32x4*>(in.data + token * in.token_stride +
                                               head[i] * in.head_stride + channel);
  }
  Angles angles = {};
  if (p.rotation.rot && channel < p.rotation.rot)
    angles = load_angles<D>(p.rotation, position, p.tokens, token, channel);
  int64_t page = -1;
  int row = 0;
  if constexpr (kAppend) {
    if (slot >= 0 && slot < int64_t(p.cache.pages) << p.cache.page_shift) {
      page = slot >> p.cache.page_shift;
      row = int(slot & ((1 << p.cache.page_shift) - 1));
    }
  }

#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int group = first + i;
    if (group >= groups) return;
    const bool is_q = group < q_groups, is_k = !is_q && group < q_groups + k_groups;
    float x[8];
    unpack8(raw[i], x);
    if (is_q || is_k) {
      const float* weight = is_q ? p.q_weight : p.k_weight;
      if (weight) norm8<D>(x, weight + channel, p.eps);
      if (p.rotation.rot) rotate8<D>(x, angles, p.rotation, lane, channel);
    }
    if (is_q || !kAppend) {
      const HeadsView& out = is_q ? p.q_out : p.k_out;
      if (live[i])
        *reinterpret_cast<u32x4*>(out.data + token * out.token_stride +
                                  head[i] * out.head_stride + channel) = pack8(x);
    } else {
      store_fp4<D>(x, is_k ? p.cache.k : p.cache.v, page,
                   (head[i] << p.cache.page_shift) + row, channel, live[i] && page >= 0);
    }
  }
}

template <int D>
hipError_t launch_dim(const NormRopeArgs& args, bool append, hipStream_t stream) {
  const NormRopeGrid grid = norm_rope_grid(args.tokens, args.q.heads, args.k.heads, D, append);
  auto launch = [&](auto kernel) {
    kernel<<<uint32_t(grid.workgroups), kNormThreads, 0, stream>>>(args, grid.q_groups, grid.k_groups,
                                                                   grid.groups, grid.chunks);
  };
  if (grid.per_wave == 4)
    launch(append ? norm_rope_kernel<D, true, 4> : norm_rope_kernel<D, false, 4>);
  else
    launch(append ? norm_rope_kernel<D, true, 1> : norm_rope_kernel<D, false, 1>);
  return hipGetLastError();
}

// One lane for 8 channels of a row, keys and values both.
template <int D>
__global__ void __launch_bounds__(kUnpackThreads)
    unpack_fp4_kernel(const Fp4CacheView cache, const int64_t* __restrict__ slots,
                      uint16_t* __restrict__ k, uint16_t* __restrict__ v, int64_t packs) {
  const int64_t index = int64_t(blockIdx.x) * kUnpackThreads + threadIdx.x;
  if (index >= packs) return;
  const int channel = int(index % (D / 8)) * 8;
  const int64_t rows = index / (D / 8);
  const int head = int(rows % cache.heads);
  const int64_t slot = slots[rows / cache.heads];
  u32x4 kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
  if (slot >= 0 && slot < int64_t(cache.pages) << cache.page_shift) {
    const int64_t page = slot >> cache.page_shift;
    const int64_t row = (int64_t(head) << cache.page_shift) +
                        (slot & ((1 << cache.page_shift) - 1));
    auto load = [&](const Fp4Rows& r) {
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(
          r.codes + page * r.code_stride + row * (D / 2) + channel / 2);
      const uint32_t byte =
          r.scales[page * r.scale_stride + row * (D / kFp4Block) + channel / kFp4Block];
      return fp4_to_bf16x8(codes, fp4_scale(byte));
    };
    kx = load(cache.k);
    vx = load(cache.v);
  }
  *reinterpret_cast<u32x4*>(k + index * 8) = kx;
  *reinterpret_cast<u32x4*>(v + index * 8) = vx;
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs& args, int dim, bool append, hipStream_t stream) {
  if (args.tokens == 0) return hipSuccess;
  switch (dim) {
    case 64: return launch_dim<64>(args, append, stream);
    case 128: return launch_dim<128>(args, append, stream);
    default: return launch_dim<256>(args, append, stream);
  }
}

hipError_t launch_unpack_fp4(const Fp4CacheView& cache, const int64_t* slots, uint16_t* k,
                             uint16_t* v, int count, int dim, hipStream_t stream) {
  const int64_t packs = int64_t(count) * cache.heads * (dim / 8);
  if (packs == 0) return hipSuccess;
  const auto kernel = dim == 64    ? unpack_fp4_kernel<64>
                      : dim == 128 ? unpack_fp4_kernel<128>
                                   : unpack_fp4_kernel<256>;
  kernel<<<uint32_t(unpack_workgroups(count, cache.heads, dim)), kUnpackThreads, 0, stream>>>(
      cache, slots, k, v, packs);
  return hipGetLastError();
}

}  // namespace ci8
