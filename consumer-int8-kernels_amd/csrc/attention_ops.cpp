// torch.ops.consumer_int8 registration of the attention operators over their C ABI
// (include/consumer_int8_attention.h; of include/consumer_int8_drafts.h what works on the same
// cache). As in torch_ops.cpp: devices, dtypes and shapes are
// checked here, geometry, alignment and overlap by the C ABI; calls run on the current stream
// of the input's device, allocate nothing and never synchronize.
#include "consumer_int8_attention.h"
#include "consumer_int8_drafts.h"
#include "torch_checks.h"

namespace {

// BF16 [tokens, heads, dim] with contiguous channels. The stride of an axis of length 1 says
// nothing and is set.
ci8_heads heads_of(const Tensor& t, int device) {
  check_type(t, ScalarType::BFloat16, device);
  STD_TORCH_CHECK(t.dim() == 3, "Expected heads [tokens, heads, dim]");
  STD_TORCH_CHECK(t.stride(2) == 1, "Heads must have contiguous channels");
  const int64_t heads = t.size(1), dim = t.size(2);
  const int64_t head_stride = heads == 1 ? dim : t.stride(1);
  return {t.data_ptr(), heads, t.size(0) <= 1 ? heads * dim : t.stride(0), head_stride};
}

const float* weight_of(const MaybeTensor& t, int64_t dim, int device) {
  if (!t.has_value()) return nullptr;
  check_plain(*t, ScalarType::Float, device);
  STD_TORCH_CHECK(t->dim() == 1 && t->size(0) == dim, "Expected FP32 norm weights [dim]");
  return static_cast<const float*>(t->data_ptr());
}

ci8_rotation rotation_of(const MaybeTensor& rope, const MaybeTensor& positions,
                         const MaybeTensor& axes, bool interleaved, int64_t tokens, int device) {
  ci8_rotation r = {};
  STD_TORCH_CHECK(rope.has_value() == positions.has_value() &&
                      (rope.has_value() || !axes.has_value()),
                  "The rotation takes a table and positions together");
  if (!rope.has_value()) return r;
  check_plain(*rope, ScalarType::Float, device);
  check_plain(*positions, ScalarType::Long, device);
  STD_TORCH_CHECK(rope->dim() == 2 && rope->size(1) > 0, "Expected an FP32 table [rows, rot]");
  const bool several = positions->dim() == 2;
  STD_TORCH_CHECK((several || positions->dim() == 1) &&
                      positions->size(several ? 1 : 0) == tokens,
                  "Expected INT64 positions [tokens] or [axes, tokens]");
  r.table = static_cast<const float*>(rope->data_ptr());
  r.rows = rope->size(0);
  r.rot = rope->size(1);
  r.positions = static_cast<const int64_t*>(positions->data_ptr());
  r.axes = several ? positions->size(0) : 1;
  r.interleaved = interleaved;
  if (axes.has_value()) {
    check_plain(*axes, ScalarType::Int, device);
    STD_TORCH_CHECK(axes->dim() == 1 && axes->size(0) == r.rot / 2,
                    "Expected INT32 axes [rot / 2]");
    r.axis_of = static_cast<const int32_t*>(axes->data_ptr());
  }
  STD_TORCH_CHECK(r.axes == 1 || axes.has_value(), "Several axes need axes [rot / 2]");
  return r;
}

// UINT8 [pages, heads, page_size, width], contiguous inside a page.
int64_t page_stride(const Tensor& t, int64_t width, const Tensor& like, int device) {
  check_type(t, ScalarType::Byte, device);
  STD_TORCH_CHECK(t.dim() == 4 && like.dim() == 4 && t.size(0) == like.size(0) &&
                      t.size(1) == like.size(1) && t.size(2) == like.size(2) &&
                      t.size(3) == width,
                  "Expected cache codes [pages, heads, page_size, dim / 2] and scales [pages, "
                  "heads, page_size, dim / 32]");
  const int64_t page = t.size(2) * width;
  STD_TORCH_CHECK(t.stride(3) == 1 && (t.size(2) == 1 || t.stride(2) == width) &&
                      (t.size(1) == 1 || t.stride(1) == page),
                  "Cache pages must be contiguous");
  return t.size(0) == 1 ? t.size(1) * page : t.stride(0);
}

ci8_fp4_cache cache_of(const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes,
                       const Tensor& v_scales, int64_t dim, int device) {
  ci8_fp4_cache c = {};
  c.k_code_page_stride = page_stride(k_codes, dim / 2, k_codes, device);
  c.k_scale_page_stride = page_stride(k_scales, dim / 32, k_codes, device);
  c.v_code_page_stride = page_stride(v_codes, dim / 2, k_codes, device);
  c.v_scale_page_stride = page_stride(v_scales, dim / 32, k_codes, device);
  c.k_codes = static_cast<uint8_t*>(k_codes.data_ptr());
  c.k_scales = static_cast<uint8_t*>(k_scales.data_ptr());
  c.v_codes = static_cast<uint8_t*>(v_codes.data_ptr());
  c.v_scales = static_cast<uint8_t*>(v_scales.data_ptr());
  c.pages = k_codes.size(0);
  c.heads = k_codes.size(1);
  c.page_size = k_codes.size(2);
  return c;
}

void check_like(const Tensor& out, const Tensor& in) {
  STD_TORCH_CHECK(out.dim() == 3 && out.size(0) == in.size(0) && out.size(1) == in.size(1) &&
                      out.size(2) == in.size(2),
                  "Outputs must have their inputs' shapes");
}

void check_tokens(const Tensor& a, const Tensor& b) {
  STD_TORCH_CHECK(a.size(0) == b.size(0) && a.size(2) == b.size(2),
                  "Heads must agree in tokens and channels");
}

void qk_norm_rope(Tensor q, Tensor k, MaybeTensor q_weight, MaybeTensor k_weight,
                  MaybeTensor rope, MaybeTensor positions, MaybeTensor axes, Tensor q_out,
                  Tensor k_out, double eps, bool interleaved) {
  const int device = q.get_device_index();
  const ci8_heads qv = heads_of(q, device), kv = heads_of(k, device);
  check_tokens(q, k);
  const ci8_heads qo = heads_of(q_out, device), ko = heads_of(k_out, device);
  check_like(q_out, q);
  check_like(k_out, k);
  const int64_t tokens = q.size(0), dim = q.size(2);
  const ci8_head_norm norm = {weight_of(q_weight, dim, device), weight_of(k_weight, dim, device),
                              eps};
  const ci8_rotation rotation =
      rotation_of(rope, positions, axes, interleaved, tokens, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_qk_norm_rope(&qv, &kv, &qo, &ko, &norm, &rotation, tokens, dim,
                                  stream_for(device)));
}

void append_fp4(MaybeTensor q, Tensor k, Tensor v, MaybeTensor q_weight, MaybeTensor k_weight,
                MaybeTensor rope, MaybeTensor positions, MaybeTensor axes, Tensor slots,
                MaybeTensor q_out, Tensor k_codes, Tensor k_scales, Tensor v_codes,
                Tensor v_scales, double eps, bool interleaved) {
  const int device = k.get_device_index();
  const ci8_heads kv = heads_of(k, device), vv = heads_of(v, device);
  check_tokens(k, v);
  STD_TORCH_CHECK(q.has_value() == q_out.has_value(), "Queries need an output, and no more");
  ci8_heads qv = {}, qo = {};
  if (q.has_value()) {
    qv = heads_of(*q, device);
    check_tokens(*q, k);
    qo = heads_of(*q_out, device);
    check_like(*q_out, *q);
  }
  check_plain(slots, ScalarType::Long, device);
  const int64_t tokens = k.size(0), dim = k.size(2);
  STD_TORCH_CHECK(slots.dim() == 1 && slots.size(0) == tokens, "Expected INT64 slots [tokens]");
  const ci8_head_norm norm = {weight_of(q_weight, dim, device), weight_of(k_weight, dim, device),
                              eps};
  const ci8_rotation rotation =
      rotation_of(rope, positions, axes, interleaved, tokens, device);
  const ci8_fp4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, dim, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_append_fp4(q.has_value() ? &qv : nullptr, &kv, &vv,
                                q.has_value() ? &qo : nullptr, &norm, &rotation,
                                static_cast<const int64_t*>(slots.data_ptr()), &cache, tokens,
                                dim, stream_for(device)));
}

void unpack_fp4(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor slots,
                Tensor k, Tensor v) {
  const int device = k.get_device_index();
  check_plain(k, ScalarType::BFloat16, device);
  check_plain(v, ScalarType::BFloat16, device);
  check_plain(slots, ScalarType::Long, device);
  STD_TORCH_CHECK(k.dim() == 3 && slots.dim() == 1 && slots.size(0) == k.size(0) &&
                      k_codes.dim() == 4 && k.size(1) == k_codes.size(1),
                  "Expected INT64 slots [count] and BF16 k, v [count, heads, dim]");
  check_like(v, k);
  const int64_t count = k.size(0), dim = k.size(2);
  const ci8_fp4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, dim, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_unpack_fp4(&cache, static_cast<const int64_t*>(slots.data_ptr()),
                                k.data_ptr(), v.data_ptr(), count, dim, stream_for(device)));
}

// Attention of chains of queries, and of trees where there are parents.
void attend(const Tensor& q, const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes,
            const Tensor& v_scales, const Tensor& page_table, const Tensor& context_lens,
            const MaybeTensor& q_starts, const Tensor* parents, const Tensor& workspace,
            const Tensor& out, const MaybeTensor& lse, double scale, int64_t max_q,
            int64_t window) {
  const int device = q.get_device_index();
  const ci8_heads qv = heads_of(q, device);
  const int64_t tokens = q.size(0), dim = q.size(2);
  const ci8_fp4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, dim, device);
  check_plain(page_table, ScalarType::Int, device);
  check_plain(context_lens, ScalarType::Int, device);
  STD_TORCH_CHECK(page_table.dim() == 2 && context_lens.dim() == 1 &&
                      context_lens.size(0) == page_table.size(0),
                  "Expected INT32 page_table [seqs, width] and context_lens [seqs]");
  const int64_t seqs = page_table.size(0);
  if (q_starts.has_value()) {
    check_plain(*q_starts, ScalarType::Int, device);
    STD_TORCH_CHECK(q_starts->dim() == 1 && q_starts->size(0) == seqs + 1,
                    "Expected INT32 q_starts [seqs + 1]");
  }
  check_plain(workspace, ScalarType::Float, device);
  STD_TORCH_CHECK(workspace.numel() >= 65536 * (dim + 2),
                  "Expected an FP32 workspace [65536, dim + 2]");
  check_plain(out, ScalarType::BFloat16, device);
  check_like(out, q);
  if (lse.has_value()) {
    check_plain(*lse, ScalarType::Float, device);
    STD_TORCH_CHECK(lse->dim() == 2 && lse->size(0) == tokens && lse->size(1) == q.size(1),
                    "Expected FP32 lse [tokens, heads]");
  }
  if (parents) {
    check_plain(*parents, ScalarType::Int, device);
    STD_TORCH_CHECK(parents->dim() == 1 && parents->size(0) == tokens,
                    "Expected INT32 parents [tokens]");
  }
  torch::stable::accelerator::DeviceGuard guard(device);
  const auto* table = static_cast<const int32_t*>(page_table.data_ptr());
  const auto* lens = static_cast<const int32_t*>(context_lens.data_ptr());
  const auto* starts =
      q_starts.has_value() ? static_cast<const int32_t*>(q_starts->data_ptr()) : nullptr;
  float* const sums = lse.has_value() ? static_cast<float*>(lse->data_ptr()) : nullptr;
  void* const stream = stream_for(device);
  raise_on_error(
      parents ? ci8_attention_fp4_tree(&qv, &cache, table, page_table.size(1), lens, starts,
                                       static_cast<const int32_t*>(parents->data_ptr()), seqs,
                                       tokens, dim, workspace.data_ptr(), out.data_ptr(), sums,
                                       scale, max_q, window, stream)
              : ci8_attention_fp4(&qv, &cache, table, page_table.size(1), lens, starts, seqs, tokens,
                                  dim, workspace.data_ptr(), out.data_ptr(), sums, scale, max_q,
                                  window, stream));
}

void attention_fp4(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales,
                   Tensor page_table, Tensor context_lens, MaybeTensor q_starts,
                   Tensor workspace, Tensor out, MaybeTensor lse, double scale, int64_t max_q,
                   int64_t window) {
  attend(q, k_codes, k_scales, v_codes, v_scales, page_table, context_lens, q_starts, nullptr,
         workspace, out, lse, scale, max_q, window);
}

void attention_fp4_tree(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales,
                        Tensor page_table, Tensor context_lens, Tensor q_starts, Tensor parents,
                        Tensor workspace, Tensor out, MaybeTensor lse, double scale, int64_t max_q,
                        int64_t window) {
  attend(q, k_codes, k_scales, v_codes, v_scales, page_table, context_lens, q_starts, &parents,
         workspace, out, lse, scale, max_q, window);
}

void move_fp4(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor rows,
              Tensor slots, Tensor q_starts) {
  const int device = rows.get_device_index();
  check_plain(rows, ScalarType::Int, device);
  check_plain(slots, ScalarType::Long, device);
  check_plain(q_starts, ScalarType::Int, device);
  STD_TORCH_CHECK(rows.dim() == 1 && slots.dim() == 1 && slots.size(0) == rows.size(0) &&
                      q_starts.dim() == 1 && q_starts.size(0) >= 1 && k_codes.dim() == 4,
                  "Expected INT32 rows [tokens], INT64 slots [tokens] and INT32 q_starts [seqs + 1]");
  const int64_t dim = k_codes.size(3) * 2;
  const ci8_fp4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, dim, device);
  torch::stable::accelerator::DeviceGuard guard(device);
  raise_on_error(ci8_move_fp4(&cache, static_cast<const int32_t*>(rows.data_ptr()),
                              static_cast<const int64_t*>(slots.data_ptr()),
                              static_cast<const int32_t*>(q_starts.data_ptr()),
                              q_starts.size(0) - 1, rows.size(0), dim, stream_for(device)));
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(consumer_int8, m) {
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? rope, Tensor? positions, Tensor? axes, Tensor(a!) q_out, Tensor(b!) k_out, float eps=1e-06, bool interleaved=False) -> ()");
  m.def("append_fp4(Tensor? q, Tensor k, Tensor v, Tensor? q_weight, Tensor? k_weight, Tensor? rope, Tensor? positions, Tensor? axes, Tensor slots, Tensor(a!)? q_out, Tensor(b!) k_codes, Tensor(c!) k_scales, Tensor(d!) v_codes, Tensor(e!) v_scales, float eps=1e-06, bool interleaved=False) -> ()");
  m.def("unpack_fp4(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor slots, Tensor(a!) k, Tensor(b!) v) -> ()");
  m.def("attention_fp4(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor page_table, Tensor context_lens, Tensor? q_starts, Tensor(a!) workspace, Tensor(b!) out, Tensor(c!)? lse, float scale, int max_q=1, int window=0) -> ()");
  m.def("attention_fp4_tree(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor page_table, Tensor context_lens, Tensor q_starts, Tensor parents, Tensor(a!) workspace, Tensor(b!) out, Tensor(c!)? lse, float scale, int max_q, int window=0) -> ()");
  m.def("move_fp4(Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, Tensor rows, Tensor slots, Tensor q_starts) -> ()");
}

STABLE_TORCH_LIBRARY_IMPL(consumer_int8, CUDA, m) {
  m.impl("qk_norm_rope", TORCH_BOX(&qk_norm_rope));
  m.impl("append_fp4", TORCH_BOX(&append_fp4));
  m.impl("unpack_fp4", TORCH_BOX(&unpack_fp4));
  m.impl("attention_fp4", TORCH_BOX(&attention_fp4));
  m.impl("attention_fp4_tree", TORCH_BOX(&attention_fp4_tree));
  m.impl("move_fp4", TORCH_BOX(&move_fp4));
}
