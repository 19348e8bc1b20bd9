// The C ABI of the attention operators (include/consumer_int8_attention.h): argument
// validation, then the launch. Pure host code up to the launch.
#include "consumer_int8_attention.h"

#include <cfloat>
#include <climits>
#include <cmath>

#include "abi_checks.h"
#include "attention_launch.h"
#include "attention_plan.h"

namespace {

using ci8::abi_fail;
using ci8::abi_launched;
using ci8::aligned;
using ci8::as_stream;
using ci8::overlap;

constexpr int64_t kMaxExtent = int64_t(1) << 46;  // bytes; far past any buffer of a GPU
// Where a page begins is held in 32 bits, in 16 bytes of codes and 8 of scales.
constexpr int64_t kMaxCacheExtent = int64_t(1) << 35;
using i128 = __int128;

bool dim_ok(int64_t dim) { return dim == 64 || dim == 128 || dim == 256; }

// Bytes from the first to past the last value of a view; -1 if over kMaxExtent.
int64_t extent(const ci8_heads& v, int64_t tokens, int64_t dim) {
  if (tokens == 0) return 0;
  const i128 last = i128(tokens - 1) * v.token_stride + i128(v.heads - 1) * v.head_stride + dim;
  return last * 2 > kMaxExtent ? -1 : int64_t(last) * 2;
}

int check_heads(const ci8_heads* v, int64_t tokens, int64_t dim) {
  if (!v) return abi_fail(CI8_ERR_GEOMETRY, "Missing heads");
  if (!(v->heads > 0 && v->heads <= 65535 && v->token_stride >= 0 && v->head_stride >= 0))
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid heads: expected 1..65535 heads and strides >= 0");
  if (v->token_stride % 8 || v->head_stride % 8 || !aligned(v->data, 16))
    return abi_fail(CI8_ERR_ALIGNMENT,
                    "Heads require 16-byte aligned data and strides that are multiples of 8");
  if (extent(*v, tokens, dim) < 0) return abi_fail(CI8_ERR_TOO_LARGE, "Heads too large");
  return CI8_OK;
}

// Rows and heads of an output must not share elements.
int check_distinct(const ci8_heads& v, int64_t tokens, int64_t dim) {
  const bool heads_apart = v.heads == 1 || v.head_stride >= dim;
  const int64_t span = (v.heads - 1) * v.head_stride + dim;
  const bool tokens_apart = tokens <= 1 || v.token_stride >= span ||
                            (v.token_stride >= dim &&
                             v.head_stride >= (tokens - 1) * v.token_stride + dim);
  if (heads_apart && tokens_apart) return CI8_OK;
  return abi_fail(CI8_ERR_OVERLAP, "Output heads overlap each other");
}

bool same(const ci8_heads& a, const ci8_heads& b) {
  return a.data == b.data && a.heads == b.heads && a.token_stride == b.token_stride &&
         a.head_stride == b.head_stride;
}

// Whether two views share elements: exact for rows of one buffer, and for heads that take turns in
// it ([tokens, heads, 3, dim]); else by their extents.
bool share(const ci8_heads& a, const ci8_heads& b, int64_t tokens, int64_t dim) {
  if (!overlap(a.data, extent(a, tokens, dim), b.data, extent(b, tokens, dim))) return false;
  if (a.head_stride == b.head_stride && a.head_stride > 0 &&
      (tokens == 1 ||
       (a.token_stride % a.head_stride == 0 && b.token_stride % b.head_stride == 0))) {
    // All heads of one view begin the same number of bytes into a stride.
    const int64_t turn = a.head_stride * 2;
    const int64_t apart = reinterpret_cast<intptr_t>(b.data) - reinterpret_cast<intptr_t>(a.data);
    const int64_t shift = ((apart % turn) + turn) % turn;
    if (shift >= dim * 2 && shift + dim * 2 <= turn) return false;
  }
  const int64_t stride = a.token_stride * 2;
  if (a.token_stride != b.token_stride || stride == 0) return true;
  const int64_t row_a = ((a.heads - 1) * a.head_stride + dim) * 2;
  const int64_t row_b = ((b.heads - 1) * b.head_stride + dim) * 2;
  if (row_a > stride || row_b > stride) return true;
  const int64_t apart = reinterpret_cast<intptr_t>(b.data) - reinterpret_cast<intptr_t>(a.data);
  const int64_t shift = ((apart % stride) + stride) % stride;
  return shift < row_a || shift + row_b > stride;
}

// Whether a view and a plain buffer share bytes, by the view's extent.
bool share(const ci8_heads& a, int64_t tokens, int64_t dim, const void* p, int64_t bytes) {
  return p && overlap(a.data, extent(a, tokens, dim), p, bytes);
}

int check_norm(const ci8_head_norm* n) {
  if (!n) return abi_fail(CI8_ERR_GEOMETRY, "Missing norm");
  if (!aligned(n->q_weight, 16) || !aligned(n->k_weight, 16))
    return abi_fail(CI8_ERR_ALIGNMENT, "Norm weights must be 16-byte aligned");
  if (!(n->eps >= 0 && std::isfinite(float(n->eps))))
    return abi_fail(CI8_ERR_GEOMETRY, "Invalid norm: eps must be finite and not negative");
  return CI8_OK;
}

int check_rotation(const ci8_rotation* r, int64_t tokens, int64_t dim) {
  if (!r) return abi_fail(CI8_ERR_GEOMETRY, "Missing rotation");
  if (r->rot == 0) return CI8_OK;
  if (!(r->rot > 0 && r->rot <= dim && r->rot % 16 == 0 && r->rows > 0 && r->axes >= 1 &&
        r->axes <= 16 && r->table && (r->positions || tokens == 0) && (r->axes == 1 || r->axis_of)))
    return abi_fail(CI8_ERR_GEOMETRY,
                    "Invalid rotation: expected 16 <= rot <= dim in steps of 16, a table, "
                    "positions, and an axis for each pair where there are several");
  if (!aligned(r->table, 16) || !aligned(r->positions, 8) || !aligned(r->axis_of, 4))
    return abi_fail(CI8_ERR_ALIGNMENT, "Rotation requires aligned buffers");
  if (i128(r->rows) * r->rot * 4 > kMaxExtent)
    return abi_fail(CI8_ERR_TOO_LARGE, "Rotation table too large");
  return CI8_OK;
}

struct Extents {
  int64_t code, scale;  // bytes of a page
  int64_t bytes[4];     // of k_codes, k_scales, v_codes, v_scales
};

int check_cache(const ci8_fp4_cache* c, int64_t dim, Extents& e) {
  if (!c) return abi_fail(CI8_ERR_GEOMETRY, "Missing cache");
  if (!(c->pages > 0 && c->pages <= INT_MAX && c->heads > 0 && c->heads <= 65535 &&
        c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0))
    return abi_fail(CI8_ERR_GEOMETRY,
                    "Invalid cache: expected pages > 0, 1..65535 heads and a page size that is "
                    "a power of two in 16..1024");
  e.code = c->heads * c->page_size * (dim / 2);
  e.scale = c->heads * c->page_size * (dim / 32);
  const int64_t strides[4] = {c->k_code_page_stride, c->k_scale_page_stride,
                              c->v_code_page_stride, c->v_scale_page_stride};
  const void* data[4] = {c->k_codes, c->k_scales, c->v_codes, c->v_scales};
  for (int i = 0; i < 4; ++i) {
    const int64_t page = i % 2 ? e.scale : e.code, unit = i % 2 ? 8 : 16;
    if (c->pages > 1 && strides[i] < page)
      return abi_fail(CI8_ERR_GEOMETRY, "Invalid cache: pages overlap");
    if (!aligned(data[i], unit) || strides[i] % unit)
      return abi_fail(CI8_ERR_ALIGNMENT,
                      "The cache requires codes on 16 and scales on 8 bytes, pages too");
    const i128 bytes = i128(c->pages - 1) * strides[i] + page;
    if (bytes > kMaxCacheExtent) return abi_fail(CI8_ERR_TOO_LARGE, "Cache too large");
    e.bytes[i] = int64_t(bytes);
  }
  return CI8_OK;
}

// Two strided runs of `rows` pages, interleaved in one buffer (as keys and values of one
// page pool are) or apart.
bool pages_share(const void* a, int64_t page_a, int64_t bytes_a, const void* b, int64_t page_b,
                 int64_t bytes_b, int64_t stride_a, int64_t stride_b) {
  if (!overlap(a, bytes_a, b, bytes_b)) return false;
  if (stride_a != stride_b || stride_a == 0) return true;
  const int64_t apart = reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a);
  const int64_t shift = ((apart % stride_a) + stride_a) % stride_a;
  return shift < page_a || shift + page_b > stride_a;
}

int check_cache_written(const ci8_fp4_cache& c, const Extents& e) {
  const void* data[4] = {c.k_codes, c.k_scales, c.v_codes, c.v_scales};
  const int64_t strides[4] = {c.k_code_page_stride, c.k_scale_page_stride, c.v_code_page_stride,
                              c.v_scale_page_stride};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (pages_share(data[i], i % 2 ? e.scale : e.code, e.bytes[i], data[j],
                      j % 2 ? e.scale : e.code, e.bytes[j], strides[i], strides[j]))
        return abi_fail(CI8_ERR_OVERLAP, "Cache buffers must not overlap");
  return CI8_OK;
}

bool shares_cache(const ci8_fp4_cache& c, const Extents& e, const void* p, int64_t bytes) {
  return overlap(c.k_codes, e.bytes[0], p, bytes) || overlap(c.k_scales, e.bytes[1], p, bytes) ||
         overlap(c.v_codes, e.bytes[2], p, bytes) || overlap(c.v_scales, e.bytes[3], p, bytes);
}

ci8::HeadsView view(const ci8_heads& v) {
  return {static_cast<uint16_t*>(v.data), int(v.heads), v.token_stride, v.head_stride};
}

ci8::RotationView view(const ci8_rotation& r) {
  return {r.table, r.positions, r.axis_of, r.rows, int(r.rot), int(r.axes), r.interleaved != 0};
}

ci8::Fp4CacheView view(const ci8_fp4_cache& c) {
  return {{c.k_codes, c.k_scales, c.k_code_page_stride, c.k_scale_page_stride},
          {c.v_codes, c.v_scales, c.v_code_page_stride, c.v_scale_page_stride},
          int(c.pages),
          int(c.heads),
          __builtin_ctzll(uint64_t(c.page_size))};
}

// An output's own checks: its geometry, its heads, and what it may share with an input.
int check_output(const ci8_heads* out, const ci8_heads& in, const ci8_head_norm& norm,
                 const ci8_rotation& r, int64_t tokens, int64_t dim) {
  if (int s = check_heads(out, tokens, dim)) return s;
  if (out->heads != in.heads)
    return abi_fail(CI8_ERR_GEOMETRY, "Outputs must have their inputs' heads");
  if (int s = check_distinct(*out, tokens, dim)) return s;
  if ((!same(*out, in) && share(*out, in, tokens, dim)) ||
      share(*out, tokens, dim, norm.q_weight, dim * 4) ||
      share(*out, tokens, dim, norm.k_weight, dim * 4) ||
      (r.rot && (share(*out, tokens, dim, r.table, r.rows * r.rot * 4) ||
                 share(*out, tokens, dim, r.positions, r.axes * tokens * 8) ||
                 share(*out, tokens, dim, r.axis_of, r.rot * 2))))
    return abi_fail(CI8_ERR_OVERLAP, "An output must be its input or overlap no input");
  return CI8_OK;
}

int check_tokens(int64_t tokens, int64_t dim) {
  if (!dim_ok(dim)) return abi_fail(CI8_ERR_GEOMETRY, "Unsupported head size: 64, 128 or 256");
  if (tokens < 0) return abi_fail(CI8_ERR_GEOMETRY, "Invalid token count");
  if (tokens > (1 << 24)) return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
  return CI8_OK;
}

// Whether the norm kernels' work-items are few enough for one launch.
int check_norm_launch(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim, bool append) {
  const ci8::NormRopeGrid grid =
      ci8::norm_rope_grid(tokens, int(q_heads), int(k_heads), int(dim), append);
  if (ci8::launch_fits(grid.workgroups, ci8::kNormThreads)) return CI8_OK;
  return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
}

}  // namespace

extern "C" {

int ci8_qk_norm_rope(const ci8_heads* q, const ci8_heads* k, const ci8_heads* q_out,
                     const ci8_heads* k_out, const ci8_head_norm* norm,
                     const ci8_rotation* rotation, int64_t tokens, int64_t dim, void* stream) {
  if (int s = check_tokens(tokens, dim)) return s;
  if (int s = check_heads(q, tokens, dim)) return s;
  if (int s = check_heads(k, tokens, dim)) return s;
  if (int s = check_norm(norm)) return s;
  if (int s = check_rotation(rotation, tokens, dim)) return s;
  if (int s = check_output(q_out, *q, *norm, *rotation, tokens, dim)) return s;
  if (int s = check_output(k_out, *k, *norm, *rotation, tokens, dim)) return s;
  if (int s = check_norm_launch(tokens, q->heads, k->heads, dim, false)) return s;
  if (share(*q_out, *k, tokens, dim) || share(*k_out, *q, tokens, dim) ||
      share(*q_out, *k_out, tokens, dim))
    return abi_fail(CI8_ERR_OVERLAP, "An output must be its input or overlap no input");
  ci8::NormRopeArgs args = {};
  args.q = view(*q);
  args.k = view(*k);
  args.q_out = view(*q_out);
  args.k_out = view(*k_out);
  args.q_weight = norm->q_weight;
  args.k_weight = norm->k_weight;
  args.eps = float(norm->eps);
  args.rotation = view(*rotation);
  args.tokens = int(tokens);
  return abi_launched(ci8::launch_norm_rope(args, int(dim), false, as_stream(stream)));
}

int ci8_append_fp4(const ci8_heads* q, const ci8_heads* k, const ci8_heads* v,
                   const ci8_heads* q_out, const ci8_head_norm* norm,
                   const ci8_rotation* rotation, const int64_t* slots,
                   const ci8_fp4_cache* cache, int64_t tokens, int64_t dim, void* stream) {
  if (int s = check_tokens(tokens, dim)) return s;
  if (int s = check_heads(k, tokens, dim)) return s;
  if (int s = check_heads(v, tokens, dim)) return s;
  if (int s = check_norm(norm)) return s;
  if (int s = check_rotation(rotation, tokens, dim)) return s;
  Extents e;
  if (int s = check_cache(cache, dim, e)) return s;
  if (k->heads != cache->heads || v->heads != cache->heads)
    return abi_fail(CI8_ERR_GEOMETRY, "Keys and values must have the cache's heads");
  if (!aligned(slots, 8)) return abi_fail(CI8_ERR_ALIGNMENT, "Slots must be 8-byte aligned");
  if (int s = check_cache_written(*cache, e)) return s;
  const ci8_heads* inputs[3] = {k, v, q};
  for (const ci8_heads* in : inputs)
    if (in && shares_cache(*cache, e, in->data, extent(*in, tokens, dim)))
      return abi_fail(CI8_ERR_OVERLAP, "The cache must not overlap an input");
  if (shares_cache(*cache, e, slots, tokens * 8) ||
      shares_cache(*cache, e, norm->q_weight, norm->q_weight ? dim * 4 : 0) ||
      shares_cache(*cache, e, norm->k_weight, norm->k_weight ? dim * 4 : 0) ||
      (rotation->rot &&
       (shares_cache(*cache, e, rotation->table, rotation->rows * rotation->rot * 4) ||
        shares_cache(*cache, e, rotation->positions, rotation->axes * tokens * 8) ||
        (rotation->axis_of && shares_cache(*cache, e, rotation->axis_of, rotation->rot * 2)))))
    return abi_fail(CI8_ERR_OVERLAP, "The cache must not overlap an input");
  ci8::NormRopeArgs args = {};
  if (q) {
    if (int s = check_heads(q, tokens, dim)) return s;
    if (int s = check_output(q_out, *q, *norm, *rotation, tokens, dim)) return s;
    if (share(*q_out, *k, tokens, dim) || share(*q_out, *v, tokens, dim) ||
        share(*q_out, tokens, dim, slots, tokens * 8) ||
        shares_cache(*cache, e, q_out->data, extent(*q_out, tokens, dim)))
      return abi_fail(CI8_ERR_OVERLAP, "An output must be its input or overlap no input");
    args.q = view(*q);
    args.q_out = view(*q_out);
  }
  if (int s = check_norm_launch(tokens, q ? q->heads : 0, k->heads, dim, true)) return s;
  args.k = view(*k);
  args.v = view(*v);
  args.q_weight = norm->q_weight;
  args.k_weight = norm->k_weight;
  args.eps = float(norm->eps);
  args.rotation = view(*rotation);
  args.slots = slots;
  args.cache = view(*cache);
  args.tokens = int(tokens);
  return abi_launched(ci8::launch_norm_rope(args, int(dim), true, as_stream(stream)));
}

int ci8_unpack_fp4(const ci8_fp4_cache* cache, const int64_t* slots, void* k, void* v,
                   int64_t count, int64_t dim, void* stream) {
  if (int s = check_tokens(count, dim)) return s;
  Extents e;
  if (int s = check_cache(cache, dim, e)) return s;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8))
    return abi_fail(CI8_ERR_ALIGNMENT, "unpack_fp4 requires aligned buffers");
  if (!ci8::launch_fits(ci8::unpack_workgroups(count, int(cache->heads), int(dim)),
                        ci8::kUnpackThreads))
    return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
  const int64_t bytes = count * cache->heads * dim * 2;
  if (overlap(k, bytes, v, bytes) || overlap(k, bytes, slots, count * 8) ||
      overlap(v, bytes, slots, count * 8) || shares_cache(*cache, e, k, bytes) ||
      shares_cache(*cache, e, v, bytes))
    return abi_fail(CI8_ERR_OVERLAP, "unpack_fp4 buffers must not overlap");
  return abi_launched(ci8::launch_unpack_fp4(view(*cache), slots, static_cast<uint16_t*>(k),
                                             static_cast<uint16_t*>(v), int(count), int(dim),
                                             as_stream(stream)));
}

int ci8_attention_fp4(const ci8_heads* q, const ci8_fp4_cache* cache,
                      const int32_t* page_table, int64_t table_width,
                      const int32_t* context_lens, const int32_t* q_starts, int64_t seqs,
                      int64_t tokens, int64_t dim, void* workspace, void* out, float* lse,
                      double scale, int64_t max_q, int64_t window, void* stream) {
  if (int s = check_tokens(tokens, dim)) return s;
  if (int s = check_heads(q, tokens, dim)) return s;
  Extents e;
  if (int s = check_cache(cache, dim, e)) return s;
  if (q->heads % cache->heads)
    return abi_fail(CI8_ERR_GEOMETRY, "Query heads must be a multiple of the cache's heads");
  if (!(seqs >= 0 && seqs <= 65535 && table_width >= 0 && max_q >= 1 && window >= 0 &&
        std::isfinite(float(scale * 1.4426950408889634)) && (q_starts || seqs == tokens)))
    return abi_fail(CI8_ERR_GEOMETRY,
                    "Invalid attention: expected at most 65535 sequences, max_q >= 1, window >= "
                    "0, a finite scale, and q_starts unless each sequence has one query");
  // Tiles of 32 tokens, of 4 row blocks each of 64 sequences, are summed in 32 bits, and up to twice
  // as many where each context takes a whole number of runs.
  if (i128(table_width) * cache->page_size > (1 << 26) - 4096 ||
      i128(seqs) * table_width * 4 > kMaxExtent)
    return abi_fail(CI8_ERR_TOO_LARGE, "Page table too large");
  if (!aligned(page_table, 4) || !aligned(context_lens, 4) || !aligned(q_starts, 4) ||
      !aligned(workspace, 16) || !aligned(out, 16) || !aligned(lse, 4))
    return abi_fail(CI8_ERR_ALIGNMENT, "attention_fp4 requires aligned buffers");
  const int64_t q_bytes = extent(*q, tokens, dim), out_bytes = tokens * q->heads * dim * 2;
  const struct {
    const void* p;
    int64_t bytes;
  } outputs[3] = {{out, out_bytes},
                  {lse, lse ? tokens * q->heads * 4 : 0},
                  {workspace, ci8::kAttentionWorkspaceRows * (dim + 2) * 4}},
    inputs[4] = {{q->data, q_bytes},
                 {page_table, seqs * table_width * 4},
                 {context_lens, seqs * 4},
                 {q_starts, q_starts ? (seqs + 1) * 4 : 0}};
  for (int i = 0; i < 3; ++i) {
    bool shared = shares_cache(*cache, e, outputs[i].p, outputs[i].bytes);
    for (const auto& in : inputs)
      shared = shared || overlap(outputs[i].p, outputs[i].bytes, in.p, in.bytes);
    for (int j = 0; j < i; ++j)
      shared = shared || overlap(outputs[i].p, outputs[i].bytes, outputs[j].p, outputs[j].bytes);
    if (shared)
      return abi_fail(CI8_ERR_OVERLAP, "attention_fp4 outputs must not overlap anything else");
  }
  if (i128(tokens) * q->heads > (i128(1) << 30))
    return abi_fail(CI8_ERR_TOO_LARGE, "Too many tokens");
  ci8::AttentionArgs args = {};
  args.q = view(*q);
  args.cache = view(*cache);
  args.page_table = page_table;
  args.context_lens = context_lens;
  args.q_starts = q_starts;
  args.workspace = static_cast<float*>(workspace);
  args.out = static_cast<uint16_t*>(out);
  args.lse = lse;
  args.scale_log2 = std::fmax(std::fabs(float(scale * 1.4426950408889634)), FLT_MIN);
  args.q_sign = scale < 0 ? 0x80008000u : 0;
  args.table_width = int(table_width);
  args.seqs = int(seqs);
  args.tokens = int(tokens);
  args.group = int(q->heads / cache->heads);
  args.max_q = int(max_q < tokens ? max_q : tokens);
  // A workgroup a unit, and one more for each of up to 256 CUs.
  if (ci8::row_split(tokens, seqs, args.group, args.max_q).prompt &&
      !ci8::launch_fits(
          ci8::prompt_units(tokens, seqs, args.group, args.max_q, args.cache.heads) + 256,
          ci8::kPromptThreads))
    return abi_fail(CI8_ERR_TOO_LARGE, "Too many sequences");
  // As many tokens as a page table holds are all; differences and sums with fewer stay in 32 bits.
  args.window = int(window < table_width * cache->page_size ? window : 0);
  return abi_launched(ci8::launch_attention_fp4(args, int(dim), as_stream(stream)));
}

}  // extern "C"
