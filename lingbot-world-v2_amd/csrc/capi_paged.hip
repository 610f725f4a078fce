// extern "C" entry points of the operators over a paged key/value cache: argument checks and launches. No allocation
// on the device and no synchronisation.

#include <string.h>

#include <algorithm>

#include "capi_checks.h"
#include "paged.h"

using namespace lbw;

namespace {

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || bytes < need))
    return fail(LBW_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need, bytes);
  return LBW_OK;
}

int fill_table(const lbw_paged_kv& c, int64_t batch, PageTable* t) {
  int shift = 0;
  while (shift < PG_MAX_SHIFT && (1 << shift) < c.page_size) ++shift;
  if (shift < PG_MIN_SHIFT || (1 << shift) != c.page_size)
    return fail(LBW_ERR_UNSUPPORTED, "page_size %d: a power of two from 16 to 1024", c.page_size);
  if (c.pages < 1) return fail(LBW_ERR_INVALID, "pages %d: a cache has one at least", c.pages);
  if (c.table_width < 0 || c.table_stride < 0)
    return fail(LBW_ERR_INVALID, "table_width %d, table_stride %lld", c.table_width, (long long)c.table_stride);
  if (batch > 0 && c.table_width > 0 && c.table == nullptr) return fail(LBW_ERR_INVALID, "table missing");
  *t = {c.table, c.table_stride, c.table_width, shift, c.pages};
  return LBW_OK;
}

int fill_page_rows(const char* name, void* p, int64_t sp, int64_t sl, int64_t sh, PageRows* r) {
  LBW_TRY(check_rows(name, p, 1, sl, sh, true));
  if (!mult8(sp) || sp < 0) return fail(LBW_ERR_INVALID, "%s: the page stride must be a multiple of 8 elements", name);
  *r = {static_cast<uint16_t*>(p), sp, sl, sh};
  return LBW_OK;
}
int fill_cache(const lbw_paged_kv& c, PageRows* k, PageRows* v) {
  LBW_TRY(fill_page_rows("the cache's k", c.k, c.k_stride_p, c.k_stride_l, c.k_stride_h, k));
  return fill_page_rows("the cache's v", c.v, c.v_stride_p, c.v_stride_l, c.v_stride_h, v);
}

// One query token per sequence: head counts, batch, q, table and lengths.
template <typename Params, typename Args>
int fill_queries(const Params* p, Args* a) {
  if (p == nullptr) return fail(LBW_ERR_INVALID, "params is NULL");
  memset(a, 0, sizeof(*a));
  if (p->batch < 0) return fail(LBW_ERR_INVALID, "batch %d", p->batch);
  if (p->head_dim != 128) return fail(LBW_ERR_UNSUPPORTED, "head_dim %d: only 128", p->head_dim);
  LBW_TRY(check_heads(p->q_heads, p->k_heads));
  LBW_TRY(check_rows("q", p->q, p->batch, p->q_stride_b, p->q_stride_h));
  LBW_TRY(fill_table(p->cache, p->batch, &a->pt));
  if (p->batch > 0 && p->lens == nullptr) return fail(LBW_ERR_INVALID, "lens missing");
  a->B = p->batch; a->Hq = p->q_heads; a->Hk = p->k_heads;
  a->q = {static_cast<const uint16_t*>(p->q), p->q_stride_b, p->q_stride_h};
  a->lens = p->lens;
  return LBW_OK;
}

int fill_paged(const lbw_attention_paged_params* p, PagedAttnArgs* a) {
  LBW_TRY(fill_queries(p, a));
  if (p->num_splits < 0 || p->num_splits > 128)
    return fail(LBW_ERR_INVALID, "num_splits %d not in [0, 128]", p->num_splits);
  LBW_TRY(fill_cache(p->cache, &a->k, &a->v));
  LBW_TRY(check_rows("out", p->out, p->batch, p->out_stride_b, p->out_stride_h));
  a->out = {static_cast<uint16_t*>(p->out), p->out_stride_b, p->out_stride_h};
  LBW_TRY(check_scale(p->softmax_scale, p->head_dim, &a->scale));
  a->scale_log2 = (float)((double)a->scale * kLog2e);
  a->group = a->Hq / a->Hk;
  if (p->selected != nullptr) {
    if (p->n_selected < 0 || ((int64_t)p->n_selected << a->pt.shift) > 0x7fffff00)
      return fail(LBW_ERR_INVALID, "n_selected %d pages of %d tokens", p->n_selected, p->cache.page_size);
    a->sel = p->selected;
    a->n_sel = p->n_selected;
  }
  if (p->prefix_keys < 0 || p->prefix_width < 0 || p->prefix_keys > ((int64_t)p->prefix_width << a->pt.shift) ||
      p->prefix_keys > 0x7fffff00)
    return fail(LBW_ERR_INVALID, "prefix of %lld keys in %d pages of %d", (long long)p->prefix_keys, p->prefix_width,
                p->cache.page_size);
  if (p->prefix_keys > 0) {
    if (p->prefix_table == nullptr) return fail(LBW_ERR_INVALID, "prefix_table missing");
    a->p_table = p->prefix_table;
    a->p_width = p->prefix_width;
    a->p_len = p->prefix_len;
    a->p_max = p->prefix_keys;
  }
  // (a workgroup each in the join)
  if ((int64_t)p->batch * p->q_heads > kMaxWorkgroups)
    return fail(LBW_ERR_UNSUPPORTED, "batch %d x %d heads", p->batch, p->q_heads);
  plan_paged(a, p->num_splits, num_cus());
  // (many for a prefix of many small pages: its pieces' page lists fit a workgroup's memory)
  if (workgroups(*a) > kMaxWorkgroups)
    return fail(LBW_ERR_UNSUPPORTED, "batch %d x %d heads, num_splits %d, off a prefix of %lld keys in pages of %d", p->batch,
                p->q_heads, p->num_splits, (long long)p->prefix_keys, p->cache.page_size);
  return LBW_OK;
}
size_t paged_bytes(const PagedAttnArgs& a) {
  return a.B > 0 && has_parts(a) ? (size_t)a.Hq * (size_t)all_rows(a) * (128 + 2) * sizeof(float) : 0;
}

int fill_select(const lbw_paged_select_params* p, SelectArgs* a) {
  LBW_TRY(fill_queries(p, a));
  if (p->count < 1 || p->first < 0 || p->last < 0 || (int64_t)p->first + p->last > p->count)
    return fail(LBW_ERR_INVALID, "count %d with the %d first and %d last pages", p->count, p->first, p->last);
  if (p->cache.bounds == nullptr || !aligned16(p->cache.bounds))
    return fail(LBW_ERR_INVALID, "bounds must be a 16-byte aligned device pointer");
  if (p->batch > 0 && p->selected == nullptr) return fail(LBW_ERR_INVALID, "selected missing");
  // (a workgroup for 32 pages, and one for all)
  const int64_t rows = (int64_t)p->batch * p->k_heads;
  if (rows > kMaxWorkgroups || rows > kMaxWorkgroups / (p->cache.table_width / 32 + 1))
    return fail(LBW_ERR_UNSUPPORTED, "batch %d x %d heads x %d pages", p->batch, p->k_heads, p->cache.table_width);
  a->bounds = static_cast<const uint16_t*>(p->cache.bounds);
  a->count = p->count; a->first = p->first; a->last = p->last;
  a->sel = p->selected;
  plan_select(a, num_cus());
  return LBW_OK;
}
size_t select_bytes(const SelectArgs& a) {
  return a.pt.width > a.count && a.chunk > 0 ? (size_t)a.B * a.Hk * a.pt.width * sizeof(uint64_t) : 0;
}

}  // namespace

extern "C" {

int lbw_paged_append(const lbw_paged_append_params* p, void* stream) {
  if (p == nullptr) return fail(LBW_ERR_INVALID, "params is NULL");
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  if (p->tokens < 0 || p->batch < 0) return fail(LBW_ERR_INVALID, "tokens %d, batch %d", p->tokens, p->batch);
  LBW_TRY(fill_turned_rows(p, &a));
  if (!p->norm && (p->wq != nullptr || p->wk != nullptr))
    return fail(LBW_ERR_INVALID, "weights without the norm");
  if (p->pos == nullptr && p->n_axes != 1)
    return fail(LBW_ERR_INVALID, "pos missing: rows are positions on one axis only, not on %d", p->n_axes);
  if (p->starts == nullptr && p->batch != p->tokens)
    return fail(LBW_ERR_INVALID, "%d tokens of %d sequences need starts", p->tokens, p->batch);
  if (p->tokens > 2 * kMaxWorkgroups)
    return fail(LBW_ERR_UNSUPPORTED, "tokens %d above %lld", p->tokens, (long long)(2 * kMaxWorkgroups));
  LBW_TRY(fill_table(p->cache, p->batch, &a.pt));
  LBW_TRY(fill_cache(p->cache, &a.kp, &a.vp));
  LBW_TRY(check_head_strides("the cache's k", a.kp.sh));
  LBW_TRY(check_head_strides("the cache's v", a.vp.sh));
  LBW_TRY(check_rows("v", p->v, p->tokens, p->v_stride_l, p->v_stride_h));
  LBW_TRY(check_rows("q_out", p->q_out, p->tokens, p->q_out_stride_l, p->q_out_stride_h));
  LBW_TRY(check_head_strides("v", p->v_stride_h));
  LBW_TRY(check_head_strides("q_out", p->q_out_stride_h));
  if (p->batch > 0 && p->lens == nullptr) return fail(LBW_ERR_INVALID, "lens missing");
  if (p->cache.bounds != nullptr && !aligned16(p->cache.bounds))
    return fail(LBW_ERR_INVALID, "bounds must be a 16-byte aligned device pointer");
  // (a workgroup of 256 for one token and 2 heads beside those of the tokens, or one of 512 for 2 to 16 heads, at most)
  if (p->cache.bounds != nullptr && p->tokens * (int64_t)p->k_heads > kMaxWorkgroups / 2)
    return fail(LBW_ERR_UNSUPPORTED, "tokens %d x %d heads", p->tokens, p->k_heads);
  a.B = p->batch;
  a.norm = p->norm != 0;
  a.v = {static_cast<const uint16_t*>(p->v), p->v_stride_l, p->v_stride_h};
  a.qo = {static_cast<uint16_t*>(p->q_out), p->q_out_stride_l, p->q_out_stride_h};
  a.starts = p->starts;
  a.lens = p->lens;
  a.bounds = static_cast<uint16_t*>(p->cache.bounds);
  if (p->tokens == 0 || p->batch == 0) return LBW_OK;  // (tokens of no sequence are left alone)
  const hipError_t e = launch_append(a, p->head_dim, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "paged append launch");
}

size_t lbw_attention_paged_workspace_size(const lbw_attention_paged_params* p) {
  PagedAttnArgs a;
  return fill_paged(p, &a) == LBW_OK ? paged_bytes(a) : 0;
}

int lbw_attention_paged(const lbw_attention_paged_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  PagedAttnArgs a;
  LBW_TRY(fill_paged(p, &a));
  if (a.B == 0) return LBW_OK;
  LBW_TRY(check_workspace(workspace, workspace_bytes, paged_bytes(a)));
  a.part = static_cast<float*>(workspace);
  const hipError_t e = launch_paged(a, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "paged attention launch");
}

size_t lbw_paged_select_workspace_size(const lbw_paged_select_params* p) {
  SelectArgs a;
  return fill_select(p, &a) == LBW_OK ? select_bytes(a) : 0;
}

int lbw_paged_select(const lbw_paged_select_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  SelectArgs a;
  LBW_TRY(fill_select(p, &a));
  if (a.B == 0) return LBW_OK;
  LBW_TRY(check_workspace(workspace, workspace_bytes, select_bytes(a)));
  a.score = static_cast<uint64_t*>(workspace);
  const hipError_t e = launch_select(a, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "page selection launch");
}

}  // extern "C"
