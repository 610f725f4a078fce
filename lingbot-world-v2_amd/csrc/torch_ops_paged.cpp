// torch.ops.lbw: the operators over a paged key/value cache (append, page selection, attention of one query token per
// sequence) over the C ABI, with their shapes for tracing. As in torch_ops.cpp every op runs on its tensors' device,
// on torch's current stream there, checks what it reads and writes, and raises RuntimeError with the library's message.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include <cstring>

#include "lbw_attn.h"
#include "torch_checks.h"
#include "torch_written.h"

namespace {

// A stride that some element uses (torch leaves any value in a dim of one element).
int64_t step_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void check_table(const char* name, const Tensor& t, const Tensor& like, int64_t batch) {
  check_int32(name, t, like);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == batch && (t.stride(1) == 1 || t.size(1) <= 1) && t.size(1) < (1ll << 31),
              name, " must be int32 [", batch, ", pages] with contiguous rows");
}
void check_vector(const char* name, const Tensor& t, const Tensor& like, int64_t n) {
  check_int32(name, t, like);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, " must be a contiguous int32 [", n,
              "] vector");
}

void fill_table(lbw_paged_kv& c, const Tensor& table) {
  c.table = table.data_ptr<int32_t>();
  c.table_stride = step_of(table, 0);
  c.table_width = (int32_t)table.size(1);
}

// The cache's k and v: bf16 [pages, page_size, kv heads, D] on `like`'s device with a contiguous head dim.
void fill_cache(lbw_paged_kv& c, const Tensor& k, const Tensor& v, const Tensor& like, int64_t heads, int64_t D) {
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->device() == like.device() && t->scalar_type() == at::kBFloat16 && t->dim() == 4 &&
                    t->size(2) == heads && t->size(3) == D && t->sizes() == k.sizes() && t->stride(3) == 1 &&
                    t->size(0) < (1ll << 31) && t->size(1) <= 1024,
                "the cache's k and v must be bf16 [pages, page_size, ", heads, ", ", D,
                "] on q's device, one shape, with a contiguous head dim and pages of at most 1024 tokens");
  c.k = k.data_ptr(); c.k_stride_p = step_of(k, 0); c.k_stride_l = step_of(k, 1); c.k_stride_h = step_of(k, 2);
  c.v = v.data_ptr(); c.v_stride_p = step_of(v, 0); c.v_stride_l = step_of(v, 1); c.v_stride_h = step_of(v, 2);
  c.pages = (int32_t)k.size(0);
  c.page_size = (int32_t)k.size(1);
}

void fill_bounds(lbw_paged_kv& c, const Tensor& bounds, const Tensor& like, int64_t heads, int64_t D) {
  TORCH_CHECK(bounds.device() == like.device() && bounds.scalar_type() == at::kBFloat16 && bounds.dim() == 4 &&
                  bounds.size(1) == heads && bounds.size(2) == 2 && bounds.size(3) == D && bounds.is_contiguous(),
              "the cache's bounds must be contiguous bf16 [pages, ", heads, ", 2, ", D, "] on q's device");
  c.bounds = bounds.data_ptr();
}

// ---- append

void paged_append_(const Tensor& q, const Tensor& k, const Tensor& v, const OptT& wq, const OptT& wk,
                   const Tensor& rope, at::IntArrayRef axes, bool interleaved, const OptT& pos, bool norm, double eps,
                   double q_scale, double k_scale, const Tensor& table, const Tensor& lens, const OptT& starts,
                   const Tensor& q_out, const Tensor& k_pages, const Tensor& v_pages, const OptT& bounds) {
  c10::DeviceGuard guard(q.device());
  lbw_paged_append_params p;
  std::memset(&p, 0, sizeof(p));
  fill_turned_rows(p, q, k, wq, wk, rope, axes, interleaved, norm ? eps : 0.0, q_scale, k_scale);
  if (pos.has_value()) fill_positions(p, *pos, q, (int64_t)axes.size());
  check_rows("v", v, q);
  check_rows("q_out", q_out, q);
  TORCH_CHECK(v.sizes() == k.sizes(), "v must have k's shape");
  TORCH_CHECK(q_out.sizes() == q.sizes(), "q_out must have q's shape");
  TORCH_CHECK(lens.dim() == 1 && lens.size(0) < (1ll << 31), "lens must be int32 [batch]");
  const int64_t B = lens.size(0);
  check_vector("lens", lens, q, B);
  check_table("table", table, q, B);
  if (starts.has_value()) check_vector("starts", *starts, q, B + 1);
  TORCH_CHECK(starts.has_value() || B == q.size(0), "without starts every sequence gets one token: ", q.size(0),
              " tokens, ", B, " sequences");
  fill_cache(p.cache, k_pages, v_pages, q, k.size(1), k.size(2));
  fill_table(p.cache, table);
  const Tensor none;
  const Tensor& edge = bounds.has_value() ? *bounds : none;
  if (bounds.has_value()) {
    fill_bounds(p.cache, edge, q, k.size(1), k.size(2));
    TORCH_CHECK(edge.size(0) == k_pages.size(0), "bounds of ", edge.size(0), " pages, a cache of ", k_pages.size(0));
  }
  p.q_stride_l = step_of(q, 0); p.q_stride_h = step_of(q, 1);
  p.k_stride_l = step_of(k, 0); p.k_stride_h = step_of(k, 1);
  p.v = v.data_ptr(); p.v_stride_l = step_of(v, 0); p.v_stride_h = step_of(v, 1);
  p.q_out = q_out.data_ptr(); p.q_out_stride_l = step_of(q_out, 0); p.q_out_stride_h = step_of(q_out, 1);
  p.batch = (int32_t)B;
  p.norm = norm;
  p.starts = starts.has_value() ? starts->data_ptr<int32_t>() : nullptr;
  p.lens = lens.data_ptr<int32_t>();
  check_written("q_out", q_out, &q, {&q, &k, &v, &k_pages, &v_pages, &edge});
  check_written("the cache's k", k_pages, nullptr, {&q, &k, &v, &v_pages, &edge});
  check_written("the cache's v", v_pages, nullptr, {&q, &k, &v, &edge});
  if (bounds.has_value()) check_written("bounds", edge, nullptr, {&q, &k, &v});
  check(lbw_paged_append(&p, stream_of(q)), "lbw_paged_append");
}

// ---- attention and selection

// One query token per sequence: q, its table and lengths.
template <typename Params>
void fill_queries(Params& p, const Tensor& q, const Tensor& table, const Tensor& lens, int64_t k_heads) {
  check_rows("q", q, q);
  TORCH_CHECK(q.size(0) < (1ll << 31) && q.size(1) < (1 << 30), "batch or heads too large");
  check_vector("lens", lens, q, q.size(0));
  check_table("table", table, q, q.size(0));
  p.batch = (int32_t)q.size(0);
  p.q_heads = (int32_t)q.size(1);
  p.k_heads = (int32_t)k_heads;
  p.head_dim = (int32_t)q.size(2);
  p.q = q.data_ptr(); p.q_stride_b = step_of(q, 0); p.q_stride_h = step_of(q, 1);
  p.lens = lens.data_ptr<int32_t>();
  fill_table(p.cache, table);
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void attention_paged_out(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                         const Tensor& lens, const OptT& selected, const OptT& prefix_table, const OptT& prefix_len,
                         int64_t prefix_keys, double scale, int64_t num_splits, const Tensor& out) {
  c10::DeviceGuard guard(q.device());
  lbw_attention_paged_params p;
  std::memset(&p, 0, sizeof(p));
  TORCH_CHECK(k_pages.dim() == 4, "the cache's k and v must be bf16 [pages, page_size, kv heads, D]");
  fill_queries(p, q, table, lens, k_pages.size(2));
  fill_cache(p.cache, k_pages, v_pages, q, k_pages.size(2), q.size(2));
  check_rows("out", out, q);
  TORCH_CHECK(out.sizes() == q.sizes(), "out must have q's shape");
  TORCH_CHECK(num_splits >= 0 && num_splits <= 128, "num_splits ", num_splits, " not in [0, 128]");
  if (selected.has_value()) {
    check_int32("selected", *selected, q);
    TORCH_CHECK(selected->dim() == 3 && selected->size(0) == q.size(0) && selected->size(1) == k_pages.size(2) &&
                    selected->is_contiguous() && selected->size(2) < (1ll << 31),
                "selected must be contiguous int32 [", q.size(0), ", ", k_pages.size(2), ", pages]");
    // (lists of no entries: not read, but lists)
    p.selected = selected->numel() > 0 ? selected->data_ptr<int32_t>() : lens.data_ptr<int32_t>();
    p.n_selected = (int32_t)selected->size(2);
  }
  TORCH_CHECK(prefix_table.has_value() || (!prefix_len.has_value() && prefix_keys < 0),
              "a prefix needs prefix_table, the pages of its keys");
  if (prefix_table.has_value()) {
    const int64_t n = prefix_table->dim() == 1 ? prefix_table->size(0) : -1;
    check_vector("prefix_table", *prefix_table, q, n);
    TORCH_CHECK(n < (1ll << 31) && prefix_keys <= n * p.cache.page_size, "prefix of ", prefix_keys, " keys in ", n,
                " pages of ", p.cache.page_size);
    p.prefix_table = prefix_table->data_ptr<int32_t>();
    p.prefix_width = (int32_t)n;
    p.prefix_keys = prefix_keys < 0 ? n * p.cache.page_size : prefix_keys;
    if (prefix_len.has_value()) {
      check_int32("prefix_len", *prefix_len, q);
      TORCH_CHECK(prefix_len->numel() == 1, "prefix_len must be one int32");
      p.prefix_len = prefix_len->data_ptr<int32_t>();
    }
  }
  p.out = out.data_ptr(); p.out_stride_b = step_of(out, 0); p.out_stride_h = step_of(out, 1);
  p.softmax_scale = (float)scale;
  TORCH_CHECK(scale == 0.0 || p.softmax_scale != 0.0f, "softmax_scale ", scale, " is 0 in fp32");
  p.num_splits = (int32_t)num_splits;
  check_written("out", out, nullptr, {&q, &k_pages, &v_pages});
  const size_t bytes = lbw_attention_paged_workspace_size(&p);
  const Tensor ws = workspace(bytes, q);
  check(lbw_attention_paged(&p, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)), "lbw_attention_paged");
}

Tensor attention_paged(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                       const Tensor& lens, const OptT& selected, const OptT& prefix_table, const OptT& prefix_len,
                       int64_t prefix_keys, double scale, int64_t num_splits) {
  Tensor out = at::empty(q.sizes(), q.options());
  attention_paged_out(q, k_pages, v_pages, table, lens, selected, prefix_table, prefix_len, prefix_keys, scale,
                      num_splits, out);
  return out;
}

Tensor paged_select(const Tensor& q, const Tensor& bounds, const Tensor& table, const Tensor& lens, int64_t page_size,
                    int64_t count, int64_t first, int64_t last) {
  c10::DeviceGuard guard(q.device());
  lbw_paged_select_params p;
  std::memset(&p, 0, sizeof(p));
  TORCH_CHECK(bounds.dim() == 4, "the cache's bounds must be bf16 [pages, kv heads, 2, D]");
  fill_queries(p, q, table, lens, bounds.size(1));
  fill_bounds(p.cache, bounds, q, bounds.size(1), q.size(2));
  TORCH_CHECK(bounds.size(0) < (1ll << 31) && page_size > 0 && page_size <= 1024, "bounds of too many pages, or a page_size of ",
              page_size);
  TORCH_CHECK(count >= 1 && count < (1ll << 31) && first >= 0 && last >= 0 && first <= count && last <= count - first,
              "count ", count, " with the ", first, " first and ", last, " last pages");
  p.cache.pages = (int32_t)bounds.size(0);
  p.cache.page_size = (int32_t)page_size;
  p.count = (int32_t)count; p.first = (int32_t)first; p.last = (int32_t)last;
  const Tensor sel = at::empty({q.size(0), bounds.size(1), count}, q.options().dtype(at::kInt));
  p.selected = sel.data_ptr<int32_t>();
  const size_t bytes = lbw_paged_select_workspace_size(&p);
  const Tensor ws = workspace(bytes, q);
  check(lbw_paged_select(&p, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)), "lbw_paged_select");
  return sel;
}

// ---- shapes for tracing
void paged_append__meta(const Tensor&, const Tensor&, const Tensor&, const OptT&, const OptT&, const Tensor&,
                        at::IntArrayRef, bool, const OptT&, bool, double, double, double, const Tensor&, const Tensor&,
                        const OptT&, const Tensor&, const Tensor&, const Tensor&, const OptT&) {}
Tensor attention_paged_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptT&,
                            const OptT&, const OptT&, int64_t, double, int64_t) {
  return at::empty(q.sizes(), q.options());
}
void attention_paged_out_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptT&,
                              const OptT&, const OptT&, int64_t, double, int64_t, const Tensor&) {}
Tensor paged_select_meta(const Tensor& q, const Tensor& bounds, const Tensor&, const Tensor&, int64_t, int64_t count,
                         int64_t, int64_t) {
  return at::empty({q.size(0), bounds.size(1), count}, q.options().dtype(at::kInt));
}

// ---- no gradients
void paged_append__autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v, const OptT& wq,
                            const OptT& wk, const Tensor& rope, at::IntArrayRef axes, bool interleaved,
                            const OptT& pos, bool norm, double eps, double q_scale, double k_scale,
                            const Tensor& table, const Tensor& lens, const OptT& starts, const Tensor& q_out,
                            const Tensor& k_pages, const Tensor& v_pages, const OptT& bounds) {
  const Tensor w0 = value_or_none(wq), w1 = value_or_none(wk), edge = value_or_none(bounds);
  refuse_gradients("paged_append_", {&q, &k, &v, &w0, &w1, &q_out, &k_pages, &v_pages, &edge});
  static auto op = handle<decltype(paged_append_)>("lbw::paged_append_");
  op.redispatch(ks & c10::after_autograd_keyset, q, k, v, wq, wk, rope, axes, interleaved, pos, norm, eps, q_scale,
                k_scale, table, lens, starts, q_out, k_pages, v_pages, bounds);
}

void attention_paged_out_autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k_pages,
                                  const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                                  const OptT& selected, const OptT& prefix_table, const OptT& prefix_len,
                                  int64_t prefix_keys, double scale, int64_t num_splits, const Tensor& out) {
  refuse_gradients("attention_paged with out", {&q, &k_pages, &v_pages, &out});
  static auto op = handle<decltype(attention_paged_out)>("lbw::attention_paged_out");
  op.redispatch(ks & c10::after_autograd_keyset, q, k_pages, v_pages, table, lens, selected, prefix_table, prefix_len,
                prefix_keys, scale, num_splits, out);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lbw, m) {
  m.def("paged_append_(Tensor q, Tensor k, Tensor v, Tensor? wq, Tensor? wk, Tensor rope, int[] axes, "
        "bool interleaved, Tensor? pos, bool norm, float eps, float q_scale, float k_scale, Tensor table, "
        "Tensor lens, Tensor? starts, Tensor(a!) q_out, Tensor(b!) k_pages, Tensor(c!) v_pages, "
        "Tensor(d!)? bounds) -> ()");
  m.def("attention_paged(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lens, "
        "Tensor? selected=None, Tensor? prefix_table=None, Tensor? prefix_len=None, int prefix_keys=-1, "
        "float softmax_scale=0., int num_splits=0) -> Tensor");
  m.def("attention_paged_out(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lens, Tensor? selected, "
        "Tensor? prefix_table, Tensor? prefix_len, int prefix_keys, float softmax_scale, int num_splits, "
        "Tensor(a!) out) -> ()");
  m.def("paged_select(Tensor q, Tensor bounds, Tensor table, Tensor lens, int page_size, int count, int first, "
        "int last) -> Tensor");
}

TORCH_LIBRARY_IMPL(lbw, CUDA, m) {
  m.impl("paged_append_", &paged_append_);
  m.impl("attention_paged", &attention_paged);
  m.impl("attention_paged_out", &attention_paged_out);
  m.impl("paged_select", &paged_select);
}

TORCH_LIBRARY_IMPL(lbw, Meta, m) {
  m.impl("paged_append_", &paged_append__meta);
  m.impl("attention_paged", &attention_paged_meta);
  m.impl("attention_paged_out", &attention_paged_out_meta);
  m.impl("paged_select", &paged_select_meta);
}

TORCH_LIBRARY_IMPL(lbw, Autograd, m) {
  m.impl("paged_append_", TORCH_FN(paged_append__autograd));
  m.impl("attention_paged_out", TORCH_FN(attention_paged_out_autograd));
  m.impl("attention_paged", torch::autograd::autogradNotImplementedFallback());
  m.impl("paged_select", torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(lbw, ADInplaceOrView, m) {
  LBW_COUNT_WRITES(m, paged_append_);
  LBW_COUNT_WRITES(m, attention_paged_out);
}
