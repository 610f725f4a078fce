// Argument checks shared by the C entry points of the operators on packed sequences and paged caches.
#pragma once

#include <math.h>
#include <stdint.h>

#include "capi_util.h"
#include "lbw_attn.h"
#include "packed.h"

namespace lbw {

// hipLaunchKernel's limit: fewer than 2^32 threads in a grid
constexpr int64_t kMaxWorkgroups = (int64_t(1) << 32) / 256 - 1;

// bf16 rows [n, heads, D]; n == 0: no pointer needed. `tile`: rows are copied in tiles of 64 with
// 32-bit byte offsets.
inline int check_rows(const char* name, const void* p, int64_t n, int64_t sl, int64_t sh, bool tile = false) {
  if (n > 0 && (p == nullptr || !aligned16(p)))
    return fail(LBW_ERR_INVALID, "%s must be a 16-byte aligned device pointer", name);
  if (!mult8(sl) || !mult8(sh))
    return fail(LBW_ERR_INVALID, "%s strides must be multiples of 8 elements", name);
  if (sl < 0 || sh < 0) return fail(LBW_ERR_INVALID, "%s has a negative stride", name);
  if (tile && sl >= (int64_t(1) << 31) / (64 * 2))
    return fail(LBW_ERR_UNSUPPORTED, "%s: token stride %lld exceeds %lld", name, (long long)sl,
                (long long)((int64_t(1) << 31) / (64 * 2) - 1));
  return LBW_OK;
}

// per-head norm: a lane's offset among the heads of one wave step is 32-bit
inline int check_head_strides(const char* name, int64_t sh) {
  if (sh >= (int64_t(1) << 26))
    return fail(LBW_ERR_UNSUPPORTED, "%s: head stride %lld exceeds %lld", name, (long long)sh,
                (long long)((int64_t(1) << 26) - 1));
  return LBW_OK;
}

inline int check_heads(int32_t hq, int32_t hk) {
  if (hq < 1 || hk < 1 || hq % hk != 0)
    return fail(LBW_ERR_INVALID, "k_heads %d must divide q_heads %d", hk, hq);
  return LBW_OK;
}

inline int check_scale(float s, int head_dim, float* scale) {
  if (!(s >= 0.0f) || isinf(s))
    return fail(LBW_ERR_INVALID, "softmax_scale must be positive and finite (0: 1/sqrt(head_dim))");
  // A row's exponents are taken against its reference times the scale, rounded to fp32: half a step of it is a
  // factor that all of the row's weights have in common, as long as it does not leave fp32 (a scaled score up to
  // 2^28 is off by 16 at most; at a scale of 1e8 ordinary scores gave sums of 0 and of infinity).
  if (s > 0.0f && (s < 1e-30f || s > 1e6f))
    return fail(LBW_ERR_UNSUPPORTED, "softmax_scale %g not in [1e-30, 1e6]", s);
  *scale = s > 0.0f ? s : 1.0f / sqrtf((float)head_dim);
  return LBW_OK;
}

constexpr double kLog2e = 1.4426950408889634;

#define LBW_TRY(x)                  \
  do {                              \
    const int rc_ = (x);            \
    if (rc_ != LBW_OK) return rc_;  \
  } while (0)

// Heads, weights, rotation table and the rows of q and k: what the per-head norm and the append have in common
// (`p` and `a` name these alike).
template <typename Params, typename Args>
int fill_turned_rows(const Params* p, Args* a) {
  LBW_TRY(check_heads(p->q_heads, p->k_heads));
  const int D = p->head_dim;
  if (D != 32 && D != 64 && D != 128 && D != 256)
    return fail(LBW_ERR_UNSUPPORTED, "head_dim %d: 32, 64, 128 or 256", D);
  if (p->q_heads > 32768) return fail(LBW_ERR_UNSUPPORTED, "q_heads %d above 32768", p->q_heads);
  if (!(p->eps >= 0.0f)) return fail(LBW_ERR_INVALID, "eps must not be negative");
  if (p->n_axes < 1 || p->n_axes > LBW_MAX_AXES)
    return fail(LBW_ERR_INVALID, "n_axes %d not in [1, %d]", p->n_axes, LBW_MAX_AXES);
  if (p->rope_pairs < 0 || 2 * (int64_t)p->rope_pairs > D)
    return fail(LBW_ERR_INVALID, "rope_pairs %d of head_dim %d", p->rope_pairs, D);
  int64_t sum = 0;
  for (int i = 0; i < LBW_MAX_AXES; ++i) {
    if (i < p->n_axes) {
      if (p->axis_pairs[i] < 0) return fail(LBW_ERR_INVALID, "axis_pairs[%d] is negative", i);
      sum += p->axis_pairs[i];
    }
    a->ax_end[i] = i + 1 < p->n_axes ? (int)sum : p->rope_pairs;
  }
  if (sum != p->rope_pairs)
    return fail(LBW_ERR_INVALID, "axis_pairs add up to %lld, rope_pairs is %d", (long long)sum,
                p->rope_pairs);
  if (!p->interleaved && p->rope_pairs % 8 != 0)
    return fail(LBW_ERR_UNSUPPORTED, "split halves need rope_pairs %d a multiple of 8", p->rope_pairs);
  if (p->rope_rows < 0 || p->rope_rows > 0x7fffffff)
    return fail(LBW_ERR_INVALID, "rope_rows %lld", (long long)p->rope_rows);
  if (p->rope_pairs > 0 && p->rope_rows > 0 &&
      (p->rope == nullptr || (reinterpret_cast<uintptr_t>(p->rope) & 7u)))
    return fail(LBW_ERR_INVALID, "the rotation table must be 8-byte aligned");
  if (p->w_dtype != LBW_W_BF16 && p->w_dtype != LBW_W_FP32)
    return fail(LBW_ERR_INVALID, "w_dtype %d: LBW_W_BF16 or LBW_W_FP32", p->w_dtype);
  if ((p->wq && !aligned16(p->wq)) || (p->wk && !aligned16(p->wk)))
    return fail(LBW_ERR_INVALID, "weights must be 16-byte aligned");
  LBW_TRY(check_rows("q", p->q, p->tokens, p->q_stride_l, p->q_stride_h));
  LBW_TRY(check_rows("k", p->k, p->tokens, p->k_stride_l, p->k_stride_h));
  LBW_TRY(check_head_strides("q", p->q_stride_h));
  LBW_TRY(check_head_strides("k", p->k_stride_h));
  a->T = p->tokens; a->Hq = p->q_heads; a->Hk = p->k_heads;
  a->q = {static_cast<const uint16_t*>(p->q), p->q_stride_l, p->q_stride_h};
  a->k = {static_cast<const uint16_t*>(p->k), p->k_stride_l, p->k_stride_h};
  a->wq = p->wq; a->wk = p->wk; a->w32 = p->w_dtype == LBW_W_FP32;
  a->eps = p->eps;
  a->inv_d = 1.0f / (float)D;
  a->table = reinterpret_cast<const float2*>(p->rope);
  a->P = (int)p->rope_rows; a->npairs = p->rope_pairs;
  a->naxes = p->n_axes; a->inter = p->interleaved != 0;
  a->pos = p->pos; a->pos_sl = p->pos_stride;
  a->q_scale = p->q_out_scale; a->k_scale = p->k_out_scale;
  return LBW_OK;
}

}  // namespace lbw
