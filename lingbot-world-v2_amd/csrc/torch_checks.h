// torch.ops.lbw: checks shared by the operators on packed sequences and paged caches -- what a call reads and writes,
// and whether a gradient is wanted of an operator that has none.
#pragma once

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>

#include "lbw_attn.h"

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;

inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == LBW_OK, what, " failed (status ", rc, "): ", lbw_last_error());
}

inline void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

inline void* ptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// bf16 [n, heads, D] on `like`'s device with a contiguous head dim
inline void check_rows(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the GPU, with q");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == 3 && (t.stride(2) == 1 || t.size(2) <= 1), name,
              " must be [tokens, heads, D] with a contiguous head dim");
}

inline void check_int32(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == like.device(), name,
              " must be int32 on q's device");
}

// Whether two bf16 tensors share an element, whatever their layouts. Elements i of a and j of b are one where the
// sum over the strides s of t_s s is the distance c of their first elements, t_s = i - j along the dims of that
// stride: an interval for each stride. Searched from the largest stride down, what is left of c within the
// smaller ones' reach; layouts that nest leave one or two t a stride. A search that takes long counts as shared.
inline bool may_overlap(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t bytes = reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr());
  auto reach = [](const Tensor& t) {  // bytes from the first element's to past the last one's
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
    return 2 * n;
  };
  if (bytes >= reach(a) || -bytes >= reach(b)) return false;  // (as most are: tensors of their own)
  if (bytes % 2 != 0) return true;
  struct Dim {
    int64_t s, lo, hi;        // lo <= t <= hi
    int64_t from, to;         // what this and the smaller strides add up to, at least and at most
  };
  c10::SmallVector<Dim, 8> dims;
  for (const Tensor* t : {&a, &b})
    for (int64_t d = 0; d < t->dim(); ++d) {
      const int64_t n = t->size(d) - 1, s = t->stride(d);
      if (n == 0 || s == 0) continue;
      auto at = std::find_if(dims.begin(), dims.end(), [&](const Dim& x) { return x.s == s; });
      if (at == dims.end()) at = dims.insert(dims.end(), Dim{s, 0, 0, 0, 0});
      if (t == &a) at->hi += n;
      else at->lo -= n;
    }
  std::sort(dims.begin(), dims.end(), [](const Dim& x, const Dim& y) { return x.s > y.s; });
  int64_t from = 0, to = 0;
  for (size_t i = dims.size(); i-- > 0;) {
    dims[i].from = from += dims[i].lo * dims[i].s;
    dims[i].to = to += dims[i].hi * dims[i].s;
  }
  int budget = 4096;
  auto search = [&](auto& self, size_t i, int64_t c) -> bool {
    if (i == dims.size()) return c == 0;
    if (c < dims[i].from || c > dims[i].to) return false;
    if (--budget < 0) return true;
    const int64_t s = dims[i].s, lo = i + 1 < dims.size() ? dims[i + 1].from : 0,
                  hi = i + 1 < dims.size() ? dims[i + 1].to : 0;
    // (both divisions rounded towards zero: a t too many at each end, which the next level turns down)
    const int64_t first = std::max(dims[i].lo, (c - hi) / s - 1), last = std::min(dims[i].hi, (c - lo) / s + 1);
    for (int64_t t = first; t <= last; ++t)
      if (self(self, i + 1, c - t * s)) return true;
    return false;
  };
  return search(search, 0, bytes / 2);
}

// An output that the caller gives: no two of its elements in one place, and apart from `others`, or exactly its
// own input.
inline void check_written(const char* name, const Tensor& out, const Tensor* own,
                   std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(at::has_internal_overlap(out) != at::MemOverlap::Yes, name,
              " has several elements in one place");
  for (const Tensor* t : others) {
    if (t == nullptr || !t->defined()) continue;
    if (t == own && t->data_ptr() == out.data_ptr() && t->strides() == out.strides()) continue;
    TORCH_CHECK(!may_overlap(out, *t), name, " overlaps another tensor of the call");
  }
}

// The rows of q and k, the weights and the rotation of a call, into the parameters of the per-head norm or the append,
// which name them alike.
template <typename Params>
void fill_turned_rows(Params& p, const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk, const Tensor& rope,
                      at::IntArrayRef axes, bool interleaved, double eps, double q_scale, double k_scale) {
  check_rows("q", q, q);
  check_rows("k", k, q);
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2),
              "q and k must have the same tokens and head dim");
  const int64_t D = q.size(2);
  TORCH_CHECK(wq.has_value() == wk.has_value(), "wq and wk: both or neither");
  for (const OptT* w : {&wq, &wk})
    if (w->has_value())
      TORCH_CHECK((*w)->device() == q.device() && (*w)->is_contiguous() && (*w)->numel() == D &&
                      ((*w)->scalar_type() == at::kBFloat16 || (*w)->scalar_type() == at::kFloat) &&
                      (*w)->scalar_type() == wq->scalar_type(),
                  "wq and wk must be contiguous [D] vectors, both bf16 or both fp32, on q's device");
  TORCH_CHECK(rope.device() == q.device() && rope.scalar_type() == at::kFloat && rope.dim() == 3 &&
                  rope.size(2) == 2 && rope.is_contiguous(),
              "rope must be a contiguous fp32 [rows, pairs, 2] table on q's device");
  const int64_t A = (int64_t)axes.size();
  TORCH_CHECK(A >= 1 && A <= LBW_MAX_AXES, "1 to ", LBW_MAX_AXES, " axes, got ", A);
  TORCH_CHECK(q.size(0) < (int64_t(1) << 31) && q.size(1) < (1 << 30), "too many tokens or heads");
  p.tokens = (int32_t)q.size(0);
  p.q_heads = (int32_t)q.size(1);
  p.k_heads = (int32_t)k.size(1);
  p.head_dim = (int32_t)D;
  p.q = q.data_ptr(); p.q_stride_l = q.stride(0); p.q_stride_h = q.stride(1);
  p.k = k.data_ptr(); p.k_stride_l = k.stride(0); p.k_stride_h = k.stride(1);
  p.wq = ptr(wq);
  p.wk = ptr(wk);
  p.w_dtype = wq.has_value() && wq->scalar_type() == at::kFloat ? LBW_W_FP32 : LBW_W_BF16;
  p.eps = (float)eps;
  p.rope = rope.data_ptr<float>();
  p.rope_rows = rope.size(0);
  p.rope_pairs = (int32_t)rope.size(1);
  p.n_axes = (int32_t)A;
  for (int64_t i = 0; i < A; ++i) p.axis_pairs[i] = (int32_t)axes[i];
  p.interleaved = interleaved;
  p.q_out_scale = (float)q_scale;
  p.k_out_scale = (float)k_scale;
}

// int32 positions [tokens, axes], or [tokens] for one axis
template <typename Params>
void fill_positions(Params& p, const Tensor& pos, const Tensor& q, int64_t A) {
  check_int32("pos", pos, q);
  TORCH_CHECK((pos.dim() == 2 ? pos.size(1) == A && (A == 1 || pos.stride(1) == 1)
                              : pos.dim() == 1 && A == 1) &&
                  pos.size(0) == q.size(0) && pos.stride(0) >= 0,
              "pos must be int32 [tokens, ", A, "] with contiguous rows");
  p.pos = pos.data_ptr<int32_t>();
  p.pos_stride = pos.stride(0);
}

inline bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

inline bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
inline Tensor value_or_none(const OptT& t) { return t.has_value() ? *t : Tensor(); }
inline OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

// The write forms give no gradient: with one wanted the call raises, as the tensors it writes would go on
// without it.
inline void refuse_gradients(const char* name, std::initializer_list<const Tensor*> ts) {
  bool wanted = any_grad(ts);
  for (const Tensor* t : ts) wanted = wanted || has_tangent(*t);
  TORCH_CHECK_NOT_IMPLEMENTED(!wanted, name, " is not differentiable: call it under torch.no_grad(), or with "
                              "tensors that require no gradient");
}

template <typename Sig>
auto handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

}  // namespace
