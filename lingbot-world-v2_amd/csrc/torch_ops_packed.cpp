// torch.ops.lbw: the operators on packed sequences (per-head norm + rotation, packed attention,
// single-token attention) over the C ABI, with their gradients for autograd and their shapes for
// tracing. As in torch_ops.cpp every op runs on its tensors' device, on torch's current stream there,
// checks what it reads and writes, and raises RuntimeError with the library's message.

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>
#include <limits>
#include <unordered_set>
#include <vector>

#include "lbw_attn.h"
#include "torch_written.h"

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == LBW_OK, what, " failed (status ", rc, "): ", lbw_last_error());
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void* ptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// bf16 [n, heads, D] on `like`'s device with a contiguous head dim
void check_rows(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the GPU, with q");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == 3 && (t.stride(2) == 1 || t.size(2) <= 1), name,
              " must be [tokens, heads, D] with a contiguous head dim");
}

void check_int32(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == like.device(), name,
              " must be int32 on q's device");
}

// Whether two bf16 tensors share an element, whatever their layouts. Elements i of a and j of b are one where the
// sum over the strides s of t_s s is the distance c of their first elements, t_s = i - j along the dims of that
// stride: an interval for each stride. Searched from the largest stride down, what is left of c within the
// smaller ones' reach; layouts that nest leave one or two t a stride. A search that takes long counts as shared.
bool may_overlap(const Tensor& a, const Tensor& b) {
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
void check_written(const char* name, const Tensor& out, const Tensor* own,
                   std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(at::has_internal_overlap(out) != at::MemOverlap::Yes, name,
              " has several elements in one place");
  for (const Tensor* t : others) {
    if (t == nullptr || !t->defined()) continue;
    if (t == own && t->data_ptr() == out.data_ptr() && t->strides() == out.strides()) continue;
    TORCH_CHECK(!may_overlap(out, *t), name, " overlaps another tensor of the call");
  }
}

// A gradient as the kernels read it: 16-byte rows, heads less than `head_limit` elements apart (an expanded or
// otherwise strided one is copied: its layout is the engine's choice, not the caller's).
Tensor grad_rows(const Tensor& g, int64_t head_limit) {
  const bool ok = g.stride(2) == 1 && g.stride(0) % 8 == 0 && g.stride(1) % 8 == 0 &&
                  g.stride(0) >= 0 && g.stride(1) >= 0 &&
                  (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15u) == 0 &&
                  g.stride(0) < (int64_t(1) << 31) / 128 && g.stride(1) < head_limit;
  return ok ? g : g.contiguous();
}

// ---- per-head norm + rotation

lbw_head_norm_rope_params head_norm_params(const Tensor& q, const Tensor& k, const OptT& wq,
                                           const OptT& wk, const Tensor& rope,
                                           at::IntArrayRef axes, bool interleaved,
                                           const Tensor& pos, double eps, double q_scale,
                                           double k_scale) {
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
  check_int32("pos", pos, q);
  TORCH_CHECK((pos.dim() == 2 ? pos.size(1) == A && (A == 1 || pos.stride(1) == 1)
                              : pos.dim() == 1 && A == 1) &&
                  pos.size(0) == q.size(0) && pos.stride(0) >= 0,
              "pos must be int32 [tokens, ", A, "] with contiguous rows");
  lbw_head_norm_rope_params p;
  std::memset(&p, 0, sizeof(p));
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
  p.pos = pos.data_ptr<int32_t>();
  p.pos_stride = pos.stride(0);
  p.q_out_scale = (float)q_scale;
  p.k_out_scale = (float)k_scale;
  return p;
}

void set_outs(lbw_head_norm_rope_params& p, const Tensor& qo, const Tensor& ko) {
  p.q_out = qo.data_ptr(); p.q_out_stride_l = qo.stride(0); p.q_out_stride_h = qo.stride(1);
  p.k_out = ko.data_ptr(); p.k_out_stride_l = ko.stride(0); p.k_out_stride_h = ko.stride(1);
}

std::tuple<Tensor, Tensor> head_norm_rope(const Tensor& q, const Tensor& k, const OptT& wq,
                                          const OptT& wk, const Tensor& rope,
                                          at::IntArrayRef axes, bool interleaved,
                                          const Tensor& pos, double eps, double q_scale,
                                          double k_scale) {
  c10::DeviceGuard guard(q.device());
  auto p = head_norm_params(q, k, wq, wk, rope, axes, interleaved, pos, eps, q_scale, k_scale);
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  set_outs(p, qo, ko);
  check(lbw_head_norm_rope(&p, stream_of(q)), "lbw_head_norm_rope");
  return {qo, ko};
}

void head_norm_rope_(const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk,
                     const Tensor& rope, at::IntArrayRef axes, bool interleaved,
                     const Tensor& pos, double eps, double q_scale, double k_scale,
                     const Tensor& q_out, const Tensor& k_out, const OptT& v, const OptT& v_out,
                     const OptT& rows) {
  c10::DeviceGuard guard(q.device());
  auto p = head_norm_params(q, k, wq, wk, rope, axes, interleaved, pos, eps, q_scale, k_scale);
  check_rows("q_out", q_out, q);
  TORCH_CHECK(q_out.sizes() == q.sizes(), "q_out must have q's shape");
  const int64_t T = q.size(0), Hk = k.size(1), D = q.size(2);
  // [T, Hk, D], or with rows a cache [T, capacity, Hk, D]
  auto out = [&](const Tensor& t, const char* name) {
    if (!rows.has_value()) {
      check_rows(name, t, q);
      TORCH_CHECK(t.sizes() == k.sizes(), name, " must have k's shape");
      return;
    }
    TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == at::kBFloat16 &&
                    t.dim() == 4 && t.size(0) == T && t.size(2) == Hk && t.size(3) == D &&
                    (t.stride(3) == 1),
                name, " must be a bf16 cache [", T, ", capacity, ", Hk, ", ", D,
                "] on q's device with a contiguous head dim");
    TORCH_CHECK(t.size(1) < (int64_t(1) << 31), name, ": capacity too large");
  };
  const int64_t l = rows.has_value() ? 1 : 0;
  out(k_out, "k_out");
  p.q_out = q_out.data_ptr(); p.q_out_stride_l = q_out.stride(0); p.q_out_stride_h = q_out.stride(1);
  p.k_out = k_out.data_ptr(); p.k_out_stride_l = k_out.stride(l); p.k_out_stride_h = k_out.stride(l + 1);
  TORCH_CHECK(v.has_value() == v_out.has_value(), "v and v_out: both or neither");
  const Tensor none;
  const Tensor& vv = v.has_value() ? *v : none;
  const Tensor& vo = v.has_value() ? *v_out : none;
  if (v.has_value()) {
    check_rows("v", vv, q);
    TORCH_CHECK(vv.sizes() == k.sizes(), "v must have k's shape");
    out(vo, "v_out");
    p.v = vv.data_ptr(); p.v_stride_l = vv.stride(0); p.v_stride_h = vv.stride(1);
    p.v_out = vo.data_ptr(); p.v_out_stride_l = vo.stride(l); p.v_out_stride_h = vo.stride(l + 1);
  }
  if (rows.has_value()) {
    check_int32("rows", *rows, q);
    TORCH_CHECK(rows->dim() == 1 && rows->size(0) == T && rows->is_contiguous(),
                "rows must be a contiguous int32 [tokens] vector");
    TORCH_CHECK(!v.has_value() || vo.size(1) == k_out.size(1), "k_out and v_out differ in capacity");
    p.rows = rows->data_ptr<int32_t>();
    p.row_count = (int32_t)k_out.size(1);
    p.k_out_stride_b = k_out.stride(0);
    p.v_out_stride_b = v.has_value() ? vo.stride(0) : 0;
  }
  check_written("q_out", q_out, &q, {&q, &k, &vv, &k_out, &vo});
  check_written("k_out", k_out, &k, {&q, &k, &vv, &vo});
  if (v.has_value()) check_written("v_out", vo, &vv, {&q, &k, &vv});
  check(lbw_head_norm_rope(&p, stream_of(q)), "lbw_head_norm_rope");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> head_norm_rope_bwd(
    const Tensor& dq_out_, const Tensor& dk_out_, const Tensor& q, const Tensor& k, const OptT& wq,
    const OptT& wk, const Tensor& rope, at::IntArrayRef axes, bool interleaved, const Tensor& pos,
    double eps, double q_scale, double k_scale) {
  c10::DeviceGuard guard(q.device());
  auto p = head_norm_params(q, k, wq, wk, rope, axes, interleaved, pos, eps, q_scale, k_scale);
  TORCH_CHECK(dq_out_.sizes() == q.sizes() && dk_out_.sizes() == k.sizes() &&
                  dq_out_.scalar_type() == at::kBFloat16 && dk_out_.scalar_type() == at::kBFloat16 &&
                  dq_out_.device() == q.device() && dk_out_.device() == q.device(),
              "the outputs' gradients must be bf16 of q's and k's shape on their device");
  const int64_t heads = int64_t(1) << 26;  // (the norm's kernels keep 32-bit offsets among a wave's heads)
  const Tensor dq_out = grad_rows(dq_out_, heads), dk_out = grad_rows(dk_out_, heads);
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  Tensor dwq = wq.has_value() ? at::empty_like(*wq) : at::empty({0}, q.options());
  Tensor dwk = wk.has_value() ? at::empty_like(*wk) : at::empty({0}, q.options());
  lbw_head_norm_rope_grads g;
  std::memset(&g, 0, sizeof(g));
  g.dq_out = dq_out.data_ptr(); g.dq_out_stride_l = dq_out.stride(0); g.dq_out_stride_h = dq_out.stride(1);
  g.dk_out = dk_out.data_ptr(); g.dk_out_stride_l = dk_out.stride(0); g.dk_out_stride_h = dk_out.stride(1);
  g.dq = dq.data_ptr(); g.dq_stride_l = dq.stride(0); g.dq_stride_h = dq.stride(1);
  g.dk = dk.data_ptr(); g.dk_stride_l = dk.stride(0); g.dk_stride_h = dk.stride(1);
  g.dwq = wq.has_value() ? dwq.data_ptr() : nullptr;
  g.dwk = wk.has_value() ? dwk.data_ptr() : nullptr;
  const size_t bytes = lbw_head_norm_rope_bwd_workspace_size(&p);
  Tensor ws;
  if (bytes > 0) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(lbw_head_norm_rope_bwd(&p, &g, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        "lbw_head_norm_rope_bwd");
  return {dq, dk, dwq, dwk};
}

// ---- packed attention

// A tensor without a contiguous head dim is copied: in the forward above autograd, so that its gradient finds
// the way back, and in the op itself, for calls that autograd does not see (inference mode).
Tensor unit(const Tensor& t) { return t.dim() != 3 || t.stride(2) == 1 ? t : t.contiguous(); }

// -> query items, key items, and the tile counts [q_tiles, q_tiles_max, k_tiles, k_tiles_max]
std::tuple<Tensor, Tensor, std::vector<int64_t>> packed_plan(const Tensor& q_lens,
                                                             const Tensor& k_lens, bool causal) {
  for (const Tensor* t : {&q_lens, &k_lens})
    TORCH_CHECK(t->device().is_cpu() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                    t->is_contiguous() && t->numel() == q_lens.numel() &&
                    t->numel() < (int64_t(1) << 31),
                "q_lens and k_lens must be int32 CPU vectors of one length");
  const int32_t n = (int32_t)q_lens.numel();
  const int32_t *ql = q_lens.data_ptr<int32_t>(), *kl = k_lens.data_ptr<int32_t>();
  lbw_packed_plan_info info;
  check(lbw_attention_packed_plan(n, ql, kl, causal, nullptr, 0, nullptr, 0, &info),
        "lbw_attention_packed_plan");
  Tensor qi = at::empty({info.n_q_items, LBW_PACKED_ITEM}, q_lens.options());
  Tensor ki = at::empty({info.n_k_items, LBW_PACKED_ITEM}, q_lens.options());
  if (info.n_q_items + info.n_k_items > 0)
    check(lbw_attention_packed_plan(n, ql, kl, causal, qi.data_ptr<int32_t>(), info.n_q_items,
                                    ki.data_ptr<int32_t>(), info.n_k_items, &info),
          "lbw_attention_packed_plan");
  return {qi, ki, {info.q_tiles, info.q_tiles_max, info.k_tiles, info.k_tiles_max}};
}

lbw_packed_params packed_params(const Tensor& q, const Tensor& k, const Tensor& v,
                                const Tensor& q_items, const Tensor& k_items,
                                at::IntArrayRef info, double scale) {
  check_rows("q", q, q);
  check_rows("k", k, q);
  check_rows("v", v, q);
  TORCH_CHECK(k.sizes() == v.sizes() && q.size(2) == k.size(2),
              "k and v must have one shape, and q's head dim");
  for (const Tensor* t : {&q_items, &k_items}) {
    check_int32("the plan's tables", *t, q);
    TORCH_CHECK(t->dim() == 2 && t->size(1) == LBW_PACKED_ITEM && t->is_contiguous() &&
                    t->size(0) < (int64_t(1) << 31),
                "the plan's tables must be contiguous int32 [items, ", LBW_PACKED_ITEM, "]");
  }
  TORCH_CHECK(q.size(1) < (1 << 30), "too many heads");
  lbw_packed_params p;
  std::memset(&p, 0, sizeof(p));
  p.q_heads = (int32_t)q.size(1);
  p.k_heads = (int32_t)k.size(1);
  p.head_dim = (int32_t)q.size(2);
  p.q_tokens = q.size(0);
  p.k_tokens = k.size(0);
  p.q = q.data_ptr(); p.q_stride_l = q.stride(0); p.q_stride_h = q.stride(1);
  p.k = k.data_ptr(); p.k_stride_l = k.stride(0); p.k_stride_h = k.stride(1);
  p.v = v.data_ptr(); p.v_stride_l = v.stride(0); p.v_stride_h = v.stride(1);
  p.softmax_scale = (float)scale;
  TORCH_CHECK(scale == 0.0 || p.softmax_scale != 0.0f, "softmax_scale ", scale, " is 0 in fp32");
  p.q_items = q_items.data_ptr<int32_t>();
  p.n_q_items = (int32_t)q_items.size(0);
  p.k_items = k_items.data_ptr<int32_t>();
  p.n_k_items = (int32_t)k_items.size(0);
  TORCH_CHECK(info.size() == 6, "the plan's tokens and tile counts (6 values) are wanted");
  TORCH_CHECK(q.size(0) == info[0] && k.size(0) == info[1], "the plan is for ", info[0], " query and ",
              info[1], " key rows");
  p.q_tiles = info[2];
  p.q_tiles_max = info[3];
  p.k_tiles = info[4];
  p.k_tiles_max = info[5];
  return p;
}

Tensor new_lse(const Tensor& q) {
  return at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
}

std::tuple<Tensor, Tensor> attention_packed(const Tensor& q_, const Tensor& k_, const Tensor& v_,
                                            const Tensor& q_items, const Tensor& k_items,
                                            at::IntArrayRef info, double scale, bool want_lse) {
  c10::DeviceGuard guard(q_.device());
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_);
  auto p = packed_params(q, k, v, q_items, k_items, info, scale);
  Tensor out = at::empty(q.sizes(), q.options());
  Tensor lse = want_lse ? new_lse(q) : at::empty({0}, q.options().dtype(at::kFloat));
  p.out = out.data_ptr(); p.out_stride_l = out.stride(0); p.out_stride_h = out.stride(1);
  p.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  const size_t bytes = lbw_attention_packed_workspace_size(&p);
  Tensor ws;
  if (bytes > 0) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(lbw_attention_packed_fwd(&p, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        "lbw_attention_packed_fwd");
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_packed_bwd(const Tensor& dout_, const Tensor& q_,
                                                        const Tensor& k_, const Tensor& v_,
                                                        const Tensor& out_, const Tensor& lse,
                                                        const Tensor& q_items,
                                                        const Tensor& k_items,
                                                        at::IntArrayRef info, double scale) {
  c10::DeviceGuard guard(q_.device());
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_), out = unit(out_);
  auto p = packed_params(q, k, v, q_items, k_items, info, scale);
  check_rows("out", out, q);
  TORCH_CHECK(dout_.sizes() == q.sizes() && dout_.scalar_type() == at::kBFloat16 &&
                  dout_.device() == q.device() && out.sizes() == q.sizes(),
              "dout and out must be bf16 of q's shape on its device");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.device() == q.device() && lse.dim() == 2 &&
                  lse.size(0) == q.size(1) && lse.size(1) == q.size(0) && lse.is_contiguous(),
              "lse must be the forward call's fp32 [heads, tokens]");
  const Tensor dout = grad_rows(dout_, std::numeric_limits<int64_t>::max());
  p.out = out.data_ptr(); p.out_stride_l = out.stride(0); p.out_stride_h = out.stride(1);
  p.lse = lse.data_ptr<float>();
  Tensor dq = at::empty(q.sizes(), q.options());
  Tensor dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
  lbw_packed_grads g;
  std::memset(&g, 0, sizeof(g));
  g.dout = dout.data_ptr(); g.dout_stride_l = dout.stride(0); g.dout_stride_h = dout.stride(1);
  g.dq = dq.data_ptr(); g.dq_stride_l = dq.stride(0); g.dq_stride_h = dq.stride(1);
  g.dk = dk.data_ptr(); g.dk_stride_l = dk.stride(0); g.dk_stride_h = dk.stride(1);
  g.dv = dv.data_ptr(); g.dv_stride_l = dv.stride(0); g.dv_stride_h = dv.stride(1);
  const size_t bytes = lbw_attention_packed_bwd_workspace_size(&p);
  Tensor ws;
  if (bytes > 0) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(lbw_attention_packed_bwd(&p, &g, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        "lbw_attention_packed_bwd");
  return {dq, dk, dv};
}

// ---- single-token attention

void attention_decode_out(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens,
                          double scale, int64_t num_splits, const Tensor& out) {
  c10::DeviceGuard guard(q.device());
  check_rows("q", q, q);
  check_rows("out", out, q);
  TORCH_CHECK(out.sizes() == q.sizes(), "out must have q's shape");
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->scalar_type() == at::kBFloat16 &&
                    t->dim() == 4 && t->size(0) == q.size(0) && t->size(3) == q.size(2) &&
                    t->sizes() == k.sizes() && (t->stride(3) == 1 || t->numel() == 0),
                "the caches must be bf16 [", q.size(0), ", capacity, kv heads, ", q.size(2),
                "] on q's device with a contiguous head dim");
  check_int32("lens", lens, q);
  TORCH_CHECK(lens.dim() == 1 && lens.size(0) == q.size(0) && lens.is_contiguous(),
              "lens must be a contiguous int32 [batch] vector");
  TORCH_CHECK(q.size(0) < (int64_t(1) << 31) && q.size(1) < (1 << 30), "batch or heads too large");
  TORCH_CHECK(num_splits >= 0 && num_splits <= 128, "num_splits ", num_splits, " not in [0, 128]");
  check_written("out", out, nullptr, {&q, &k, &v});
  lbw_decode_params p;
  std::memset(&p, 0, sizeof(p));
  p.batch = (int32_t)q.size(0);
  p.q_heads = (int32_t)q.size(1);
  p.k_heads = (int32_t)k.size(2);
  p.head_dim = (int32_t)q.size(2);
  p.capacity = k.size(1);
  p.q = q.data_ptr(); p.q_stride_b = q.stride(0); p.q_stride_h = q.stride(1);
  p.k = k.data_ptr(); p.k_stride_b = k.stride(0); p.k_stride_l = k.stride(1); p.k_stride_h = k.stride(2);
  p.v = v.data_ptr(); p.v_stride_b = v.stride(0); p.v_stride_l = v.stride(1); p.v_stride_h = v.stride(2);
  p.lens = lens.data_ptr<int32_t>();
  p.out = out.data_ptr(); p.out_stride_b = out.stride(0); p.out_stride_h = out.stride(1);
  p.softmax_scale = (float)scale;
  TORCH_CHECK(scale == 0.0 || p.softmax_scale != 0.0f, "softmax_scale ", scale, " is 0 in fp32");
  p.num_splits = (int32_t)num_splits;
  const size_t bytes = lbw_attention_decode_workspace_size(&p);
  Tensor ws;
  if (bytes > 0) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(lbw_attention_decode(&p, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        "lbw_attention_decode");
}

Tensor attention_decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens,
                        double scale, int64_t num_splits) {
  Tensor out = at::empty(q.sizes(), q.options());
  attention_decode_out(q, k, v, lens, scale, num_splits, out);
  return out;
}

// ---- shapes for tracing
std::tuple<Tensor, Tensor> head_norm_rope_meta(const Tensor& q, const Tensor& k, const OptT&,
                                               const OptT&, const Tensor&, at::IntArrayRef, bool,
                                               const Tensor&, double, double, double) {
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
}
void head_norm_rope__meta(const Tensor&, const Tensor&, const OptT&, const OptT&, const Tensor&,
                          at::IntArrayRef, bool, const Tensor&, double, double, double,
                          const Tensor&, const Tensor&, const OptT&, const OptT&, const OptT&) {}
std::tuple<Tensor, Tensor, Tensor, Tensor> head_norm_rope_bwd_meta(
    const Tensor&, const Tensor&, const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk,
    const Tensor&, at::IntArrayRef, bool, const Tensor&, double, double, double) {
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()),
          wq.has_value() ? at::empty_like(*wq) : at::empty({0}, q.options()),
          wk.has_value() ? at::empty_like(*wk) : at::empty({0}, q.options())};
}
std::tuple<Tensor, Tensor> attention_packed_meta(const Tensor& q, const Tensor&, const Tensor&,
                                                 const Tensor&, const Tensor&, at::IntArrayRef,
                                                 double, bool want_lse) {
  return {at::empty(q.sizes(), q.options()),
          want_lse ? new_lse(q) : at::empty({0}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor, Tensor> attention_packed_bwd_meta(
    const Tensor&, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor&, const Tensor&,
    const Tensor&, const Tensor&, at::IntArrayRef, double) {
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()),
          at::empty(v.sizes(), v.options())};
}
Tensor attention_decode_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&, double,
                             int64_t) {
  return at::empty(q.sizes(), q.options());
}
void attention_decode_out_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&, double,
                               int64_t, const Tensor&) {}

// ---- gradients

// A backward pass that is captured into a graph must not end in a leaf whose gradient node belongs to
// another stream (an eager graph of the same leaf, still alive, made it there): the engine would
// tie that stream into the capture, which ends the process. Raised here instead.
void refuse_foreign_leaves() {
  namespace ag = torch::autograd;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const c10::impl::VirtualGuardImpl impl(c10::DeviceType::CUDA);
  const c10::Stream here = impl.getStream(impl.getDevice());
  std::vector<ag::Node*> todo;
  std::unordered_set<ag::Node*> seen;
  if (const auto node = ag::get_current_node()) todo.push_back(node.get());
  while (!todo.empty()) {
    ag::Node* n = todo.back();
    todo.pop_back();
    if (!seen.insert(n).second) continue;
    if (dynamic_cast<ag::AccumulateGrad*>(n) != nullptr) {
      const auto s = n->stream();
      TORCH_CHECK(!s.has_value() || *s == here,
                  "a captured backward pass reaches a leaf that an eager graph on another stream "
                  "still holds: drop that graph (its outputs) before the capture, or detach the leaf");
    }
    for (const auto& e : n->next_edges())
      if (e.is_valid()) todo.push_back(e.function.get());
  }
}

bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// The operators have reverse-mode derivatives only: a forward-mode tangent is refused, not dropped.
void refuse_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), name, ": forward-mode derivatives are not implemented");
}

// A backward pass that builds no graph of its own calls the gradient operators below autograd (one that
// does, or that has tangents, meets autograd's entry for them, which raises: they have no derivatives).
struct BelowAutograd {
  std::optional<at::AutoDispatchBelowADInplaceOrView> guard;
  BelowAutograd(const torch::autograd::variable_list& g, const torch::autograd::variable_list& saved) {
    if (at::GradMode::is_enabled()) return;
    for (const auto* ts : {&g, &saved})
      for (const Tensor& t : *ts)
        if (has_tangent(t)) return;
    guard.emplace();
  }
};

bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
Tensor value_or_none(const OptT& t) { return t.has_value() ? *t : Tensor(); }
OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

// The write forms give no gradient: with one wanted the call raises, as the tensors it writes would go on
// without it.
void refuse_gradients(const char* name, std::initializer_list<const Tensor*> ts) {
  bool wanted = any_grad(ts);
  for (const Tensor* t : ts) wanted = wanted || has_tangent(*t);
  TORCH_CHECK_NOT_IMPLEMENTED(!wanted, name, " is not differentiable: call it under torch.no_grad(), or with "
                              "tensors that require no gradient");
}

template <typename Sig>
auto handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

auto call_head_norm(const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk,
                    const Tensor& rope, at::IntArrayRef axes, bool inter, const Tensor& pos,
                    double eps, double qs, double ks) {
  static auto op = handle<decltype(head_norm_rope)>("lbw::head_norm_rope");
  return op.call(q, k, wq, wk, rope, axes, inter, pos, eps, qs, ks);
}

struct HeadNorm : torch::autograd::Function<HeadNorm> {
  using Ctx = torch::autograd::AutogradContext;
  static torch::autograd::variable_list forward(Ctx* ctx, const Tensor& q, const Tensor& k,
                                                const OptT& wq, const OptT& wk,
                                                const Tensor& rope, std::vector<int64_t> axes,
                                                bool inter, const Tensor& pos, double eps,
                                                double qs, double ks) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [qo, ko] = call_head_norm(q, k, wq, wk, rope, axes, inter, pos, eps, qs, ks);
    ctx->save_for_backward({q, k, value_or_none(wq), value_or_none(wk), rope, pos});
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["inter"] = inter;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["qs"] = qs;
    ctx->saved_data["ks"] = ks;
    return {qo, ko};
  }
  static torch::autograd::variable_list backward(Ctx* ctx, torch::autograd::variable_list g) {
    refuse_foreign_leaves();
    const auto s = ctx->get_saved_variables();
    const BelowAutograd below(g, s);
    const Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3];
    const Tensor dq_out = g[0].defined() ? g[0] : at::zeros_like(q);
    const Tensor dk_out = g[1].defined() ? g[1] : at::zeros_like(k);
    static auto op = handle<decltype(head_norm_rope_bwd)>("lbw::head_norm_rope_bwd");
    auto [dq, dk, dwq, dwk] =
        op.call(dq_out, dk_out, q, k, opt(wq), opt(wk), s[4], ctx->saved_data["axes"].toIntVector(),
                ctx->saved_data["inter"].toBool(), s[5], ctx->saved_data["eps"].toDouble(),
                ctx->saved_data["qs"].toDouble(), ctx->saved_data["ks"].toDouble());
    const Tensor none;
    return {dq, dk, wq.defined() ? dwq : none, wk.defined() ? dwk : none,
            none, none, none, none, none, none, none};
  }
};

std::tuple<Tensor, Tensor> head_norm_rope_autograd(const Tensor& q, const Tensor& k,
                                                   const OptT& wq, const OptT& wk,
                                                   const Tensor& rope, at::IntArrayRef axes,
                                                   bool inter, const Tensor& pos, double eps,
                                                   double qs, double ks) {
  const Tensor w0 = value_or_none(wq), w1 = value_or_none(wk);
  refuse_tangents("head_norm_rope", {&q, &k, &w0, &w1});
  if (!any_grad({&q, &k, &w0, &w1})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_head_norm(q, k, wq, wk, rope, axes, inter, pos, eps, qs, ks);
  }
  auto r = HeadNorm::apply(q, k, wq, wk, rope, axes.vec(), inter, pos, eps, qs, ks);
  return {r[0], r[1]};
}

void head_norm_rope__autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const OptT& wq,
                              const OptT& wk, const Tensor& rope, at::IntArrayRef axes, bool inter,
                              const Tensor& pos, double eps, double q_scale, double k_scale, const Tensor& q_out,
                              const Tensor& k_out, const OptT& v, const OptT& v_out, const OptT& rows) {
  const Tensor w0 = value_or_none(wq), w1 = value_or_none(wk), vv = value_or_none(v), vo = value_or_none(v_out);
  refuse_gradients("head_norm_rope_", {&q, &k, &w0, &w1, &vv, &q_out, &k_out, &vo});
  static auto op = handle<decltype(head_norm_rope_)>("lbw::head_norm_rope_");
  op.redispatch(ks & c10::after_autograd_keyset, q, k, wq, wk, rope, axes, inter, pos, eps, q_scale, k_scale,
                q_out, k_out, v, v_out, rows);
}

void attention_decode_out_autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v,
                                   const Tensor& lens, double scale, int64_t num_splits, const Tensor& out) {
  refuse_gradients("attention_decode with out", {&q, &k, &v, &out});
  static auto op = handle<decltype(attention_decode_out)>("lbw::attention_decode_out");
  op.redispatch(ks & c10::after_autograd_keyset, q, k, v, lens, scale, num_splits, out);
}

auto call_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qi,
                 const Tensor& ki, at::IntArrayRef info, double scale, bool want_lse) {
  static auto op = handle<decltype(attention_packed)>("lbw::attention_packed");
  return op.call(q, k, v, qi, ki, info, scale, want_lse);
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  using Ctx = torch::autograd::AutogradContext;
  static torch::autograd::variable_list forward(Ctx* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& v, const Tensor& qi,
                                                const Tensor& ki, std::vector<int64_t> info,
                                                double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse] = call_packed(q, k, v, qi, ki, info, scale, true);
    ctx->save_for_backward({q, k, v, out, lse, qi, ki});
    ctx->saved_data["info"] = info;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static torch::autograd::variable_list backward(Ctx* ctx, torch::autograd::variable_list g) {
    refuse_foreign_leaves();
    const auto s = ctx->get_saved_variables();
    const BelowAutograd below(g, s);
    const Tensor none;
    if (!g[0].defined()) return {none, none, none, none, none, none, none};
    static auto op = handle<decltype(attention_packed_bwd)>("lbw::attention_packed_bwd");
    auto [dq, dk, dv] = op.call(g[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6],
                                ctx->saved_data["info"].toIntVector(),
                                ctx->saved_data["scale"].toDouble());
    return {dq, dk, dv, none, none, none, none};
  }
};

std::tuple<Tensor, Tensor> attention_packed_autograd(const Tensor& q_, const Tensor& k_,
                                                     const Tensor& v_, const Tensor& qi,
                                                     const Tensor& ki, at::IntArrayRef info,
                                                     double scale, bool want_lse) {
  refuse_tangents("attention_packed", {&q_, &k_, &v_});
  const Tensor q = unit(q_), k = unit(k_), v = unit(v_);
  if (!any_grad({&q, &k, &v})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_packed(q, k, v, qi, ki, info, scale, want_lse);
  }
  auto r = PackedAttention::apply(q, k, v, qi, ki, info.vec(), scale);
  return {r[0], r[1]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lbw, m) {
  m.def("head_norm_rope(Tensor q, Tensor k, Tensor? wq, Tensor? wk, Tensor rope, int[] axes, "
        "bool interleaved, Tensor pos, float eps, float q_scale, float k_scale) "
        "-> (Tensor, Tensor)");
  m.def("head_norm_rope_(Tensor q, Tensor k, Tensor? wq, Tensor? wk, Tensor rope, int[] axes, "
        "bool interleaved, Tensor pos, float eps, float q_scale, float k_scale, "
        "Tensor(a!) q_out, Tensor(b!) k_out, Tensor? v, Tensor(c!)? v_out, Tensor? rows) -> ()");
  m.def("head_norm_rope_bwd(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, Tensor? wq, "
        "Tensor? wk, Tensor rope, int[] axes, bool interleaved, Tensor pos, float eps, "
        "float q_scale, float k_scale) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("packed_plan(Tensor q_lens, Tensor k_lens, bool causal) -> (Tensor, Tensor, int[])");
  m.def("attention_packed(Tensor q, Tensor k, Tensor v, Tensor q_items, Tensor k_items, "
        "int[] info, float softmax_scale=0., bool want_lse=True) -> (Tensor, Tensor)");
  m.def("attention_packed_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, "
        "Tensor q_items, Tensor k_items, int[] info, float softmax_scale=0.) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("attention_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor lens, "
        "float softmax_scale=0., int num_splits=0) -> Tensor");
  m.def("attention_decode_out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor lens, "
        "float softmax_scale, int num_splits, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(lbw, CPU, m) { m.impl("packed_plan", &packed_plan); }

TORCH_LIBRARY_IMPL(lbw, CUDA, m) {
  m.impl("head_norm_rope", &head_norm_rope);
  m.impl("head_norm_rope_", &head_norm_rope_);
  m.impl("head_norm_rope_bwd", &head_norm_rope_bwd);
  m.impl("attention_packed", &attention_packed);
  m.impl("attention_packed_bwd", &attention_packed_bwd);
  m.impl("attention_decode", &attention_decode);
  m.impl("attention_decode_out", &attention_decode_out);
}

TORCH_LIBRARY_IMPL(lbw, Meta, m) {
  m.impl("head_norm_rope", &head_norm_rope_meta);
  m.impl("head_norm_rope_", &head_norm_rope__meta);
  m.impl("head_norm_rope_bwd", &head_norm_rope_bwd_meta);
  m.impl("attention_packed", &attention_packed_meta);
  m.impl("attention_packed_bwd", &attention_packed_bwd_meta);
  m.impl("attention_decode", &attention_decode_meta);
  m.impl("attention_decode_out", &attention_decode_out_meta);
}

TORCH_LIBRARY_IMPL(lbw, Autograd, m) {
  m.impl("head_norm_rope", &head_norm_rope_autograd);
  m.impl("attention_packed", &attention_packed_autograd);
  m.impl("head_norm_rope_", TORCH_FN(head_norm_rope__autograd));
  m.impl("attention_decode_out", TORCH_FN(attention_decode_out_autograd));
  // no second derivatives, and none through single-token attention: their backward pass raises
  m.impl("head_norm_rope_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("attention_packed_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("attention_decode", torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(lbw, ADInplaceOrView, m) {
  LBW_COUNT_WRITES(m, head_norm_rope_);
  LBW_COUNT_WRITES(m, attention_decode_out);
}
