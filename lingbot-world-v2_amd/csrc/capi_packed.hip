// extern "C" entry points of the operators on packed sequences: argument checks, the work items of
// packed attention, launches. No allocation on the device and no synchronisation.

#include <math.h>
#include <string.h>

#include <algorithm>
#include <array>
#include <new>
#include <vector>

#include "capi_checks.h"

using namespace lbw;

namespace {

// packed rows: a tile past the last one still has a 32-bit index
constexpr int64_t kMaxTokens = 0x7fffff00;

int fill_head_norm(const lbw_head_norm_rope_params* p, HeadNormArgs* a) {
  if (p == nullptr) return fail(LBW_ERR_INVALID, "params is NULL");
  memset(a, 0, sizeof(*a));
  if (p->tokens < 0) return fail(LBW_ERR_INVALID, "tokens %d", p->tokens);
  LBW_TRY(fill_turned_rows(p, a));
  if (p->tokens > 0 && p->pos == nullptr) return fail(LBW_ERR_INVALID, "pos missing");
  return LBW_OK;
}

int fill_packed(const lbw_packed_params* p, PackedArgs* a) {
  if (p == nullptr) return fail(LBW_ERR_INVALID, "params is NULL");
  memset(a, 0, sizeof(*a));
  if (p->head_dim != 128) return fail(LBW_ERR_UNSUPPORTED, "head_dim %d: only 128", p->head_dim);
  LBW_TRY(check_heads(p->q_heads, p->k_heads));
  if (p->q_tokens < 0 || p->k_tokens < 0 || p->q_tokens > kMaxTokens || p->k_tokens > kMaxTokens)
    return fail(LBW_ERR_INVALID, "q_tokens %lld, k_tokens %lld", (long long)p->q_tokens,
                (long long)p->k_tokens);
  LBW_TRY(check_rows("q", p->q, p->q_tokens, p->q_stride_l, p->q_stride_h, true));
  LBW_TRY(check_rows("k", p->k, p->k_tokens, p->k_stride_l, p->k_stride_h, true));
  LBW_TRY(check_rows("v", p->v, p->k_tokens, p->v_stride_l, p->v_stride_h, true));
  LBW_TRY(check_rows("out", p->out, p->q_tokens, p->out_stride_l, p->out_stride_h));
  float scale = 0.0f;
  LBW_TRY(check_scale(p->softmax_scale, p->head_dim, &scale));
  if (p->n_q_items < 0 || (p->n_q_items > 0 && p->q_items == nullptr))
    return fail(LBW_ERR_INVALID, "q_items missing");
  if (p->q_tiles < 0 || p->q_tiles_max < 0 || p->k_tiles < 0 || p->k_tiles_max < 0 ||
      std::max(std::max(p->q_tiles, p->q_tiles_max), std::max(p->k_tiles, p->k_tiles_max)) >
          (int64_t(1) << 56) / p->q_heads)
    return fail(LBW_ERR_INVALID, "the plan's tile counts are out of range");
  a->q = {static_cast<const uint16_t*>(p->q), p->q_stride_l, p->q_stride_h};
  a->k = {static_cast<const uint16_t*>(p->k), p->k_stride_l, p->k_stride_h};
  a->v = {static_cast<const uint16_t*>(p->v), p->v_stride_l, p->v_stride_h};
  a->out = {static_cast<uint16_t*>(p->out), p->out_stride_l, p->out_stride_h};
  a->lse = p->lse;
  a->Tq = p->q_tokens; a->Tk = p->k_tokens; a->Hq = p->q_heads; a->Hk = p->k_heads;
  a->scale = scale;
  a->scale_log2 = (float)((double)scale * kLog2e);
  a->q_items = p->q_items; a->n_q_items = p->n_q_items;
  a->k_items = p->k_items; a->n_k_items = p->n_k_items;
  return LBW_OK;
}

// How a kernel's items are cut. `slots` workgroups run at once; an item much longer than a slot's share of
// all tiles ends last. A piece costs its partial results' way to memory and back and a share of a
// second launch, some tiles of its time, so pieces are long: one and a half shares, `least` tiles
// at least (from 256 tiles a share on, where that cost is small beside an uncut item, two thirds of a share),
// and nothing is cut that would give fewer than `times` / 2 pieces. Measured, uncut / cut: forward, 256 rows over
// 4680 + 1816 + 3111 keys x 40/8 heads 83 / 70 us, 16 rows over 8192 keys 130 / 32, 5000 causal x 5/1
// 90 / 62, but 2048 causal x 40/8 (32 tiles, 21 a share) 54 / 64; gradient of 2048 x 40/8 299 / 190, 4680 x 12/4
// 446 / 295, 16384 x 16/2 4706 / 3690, but 8 x 512 x 40/8 (40 tiles, 25 a share) 131 / 185.
PackedSplit split_items(int64_t items, int64_t heads, int64_t tiles, int64_t longest, int64_t slots,
                        int64_t least, int64_t times) {
  PackedSplit s = {0, 1, 1};
  if (tiles <= 0 || longest <= 0 || items <= 0) return s;
  // Nearly equal items in up to five rounds, the last not full: as many are cut as would be in it, into pieces
  // for all slots, of 32 tiles or more (shorter ones: no gain at 25 tiles, the emptier chip clocks higher).
  // Forward, uncut / cut: 6144 full x 12/4 294 / 251 us, 1800 rows over 20000 keys x 40/8 873 / 752, 3600 over
  // 46800 3730 / 3509; gradient of 4680 over 9360 3140 / 2886.
  const int64_t units = items * heads, rest = units % slots;
  if (tiles / items >= longest - longest / 5 && units >= slots && units < 5 * slots && rest > 0) {
    const int64_t n = (rest + heads - 1) / heads;
    const int64_t c = std::min<int64_t>(std::min<int64_t>(16, slots / (n * heads)), longest / 32);
    if (c >= 2)
      return PackedSplit{(int)n, (int)c, (int)std::min<int64_t>((longest + c - 1) / c, 1 << 30)};
  }
  const int64_t share = tiles * heads / slots;
  const int64_t piece = std::max<int64_t>(least, share < 256 ? share * 3 / 2 : share * 2 / 3);
  if (2 * longest < times * piece) return s;
  s.piece = (int)std::min<int64_t>(piece, 1 << 30);
  s.smax = (int)std::min<int64_t>(16, (longest + s.piece - 1) / s.piece);
  if (s.smax < 2) return PackedSplit{0, 1, 1};
  // (the items longer than a piece come first in the table, and are no more than this)
  s.n_split = (int)std::min<int64_t>(items, std::max<int64_t>(1, tiles / s.piece));
  return s;
}
// forward and dQ: two workgroups per CU. Fewer items, more idle CUs: shorter pieces (least 16 / this rule: forward,
// 12 items 31.5 / 19.8 us, 48 31.6 / 21.5, 64 23.1 / 20.2, 120 31.4 / 27.4; of 8 / 16 with 312 38.2 / 36.6).
PackedSplit split_q(const lbw_packed_params* p) {
  return split_items(p->n_q_items, p->q_heads, p->q_tiles, p->q_tiles_max, 2 * num_cus(),
                     std::clamp<int64_t>(p->n_q_items * (int64_t)p->q_heads / 10, 8, 16), 4);
}
// dK and dV: one workgroup per CU, an item's tiles those of all heads of the group. Where items leave CUs idle
// even at two workgroups each (halves_k), a tile takes half the time and a piece costs twice as many, and pieces
// that leave no room for two workgroups each lose that half; so pieces get longer with the items (least 24 / 32 /
// 48, gradient: 16 items 57 / 66 / 89 us, 48 items 81 / 71 / 93, 64 items 90 / 97 / 88).
PackedSplit split_k(const lbw_packed_params* p) {
  const int64_t group = p->q_heads / p->k_heads;
  const int64_t units = (int64_t)p->n_k_items * p->k_heads;
  const int64_t least = 2 * units <= num_cus() ? std::clamp<int64_t>(units * 3 / 4, 24, 48) : 24;
  return split_items(p->n_k_items, p->k_heads, p->k_tiles * group, p->k_tiles_max * group, num_cus(), least, 3);
}
// Two workgroups for an item's (or a piece's) keys where that many run at once and have more than four tiles.
// Gradient, one / two: 311 + 97 + 512 + 5 x 12/4 62 / 49 us, 1024 x 16 59 / 52, 16 x 256 x 12/4 (128 items,
// 256 CUs) 53 / 48, but 5 x 60 x 12 (one tile) 18.6 / 20.2.
bool halves_k(const lbw_packed_params* p, const PackedSplit& s) {
  return 2 * (p->n_k_items + (int64_t)s.n_split * (s.smax - 1)) * p->k_heads <= num_cus() &&
         p->k_tiles_max * (p->q_heads / p->k_heads) > 4;
}
size_t part_bytes(const PackedSplit& s, int heads, int floats) {
  return (size_t)s.n_split * heads * s.smax * floats * sizeof(float);
}
int check_grid(const PackedSplit& s, int64_t items, int64_t heads, int64_t limit) {
  if (items + (int64_t)s.n_split * (s.smax - 1) > limit / heads)
    return fail(LBW_ERR_UNSUPPORTED, "%lld work items x %lld heads", (long long)items, (long long)heads);
  return LBW_OK;
}
void set_split(PackedArgs* a, const PackedSplit& s, void* part) {
  a->n_split = s.n_split;
  a->smax = s.smax;
  a->piece = s.piece;
  a->part = static_cast<float*>(part);
}
// -delta and -lse / scale of the gradient, rounded up to 16 bytes
size_t stat_bytes(const lbw_packed_params* p) {
  return (2 * (size_t)p->q_heads * (size_t)p->q_tokens * sizeof(float) + 15) / 16 * 16;
}
bool sane(const lbw_packed_params* p) {
  return p != nullptr && p->q_heads >= 1 && p->k_heads >= 1 && p->q_heads % p->k_heads == 0 &&
         p->q_tokens >= 0 && p->q_tokens <= kMaxTokens;
}

int pieces_for(const lbw_decode_params* p) {
  return decode_pieces(p->batch, p->q_heads, p->k_heads, p->capacity, p->num_splits, num_cus());
}
size_t decode_bytes(const lbw_decode_params* p, int pieces) {
  return pieces > 0 ? (size_t)p->q_heads * ((size_t)pieces + p->batch) * (p->head_dim + 2) * sizeof(float)
                    : 0;
}

int check_decode(const lbw_decode_params* p) {
  if (p == nullptr) return fail(LBW_ERR_INVALID, "params is NULL");
  if (p->batch < 0 || p->capacity < 0 || p->capacity > 0x7fffff00)
    return fail(LBW_ERR_INVALID, "batch %d, capacity %lld", p->batch, (long long)p->capacity);
  if (p->head_dim != 128) return fail(LBW_ERR_UNSUPPORTED, "head_dim %d: only 128", p->head_dim);
  LBW_TRY(check_heads(p->q_heads, p->k_heads));
  if (p->num_splits < 0 || p->num_splits > 128)
    return fail(LBW_ERR_INVALID, "num_splits %d not in [0, 128]", p->num_splits);
  const int64_t blocks = (p->q_heads / p->k_heads + 31) / 32;
  if ((int64_t)p->batch * p->k_heads * blocks * 128 > kMaxWorkgroups)
    return fail(LBW_ERR_UNSUPPORTED, "batch %d x %d heads", p->batch, p->q_heads);
  return LBW_OK;
}

using Item = std::array<int32_t, LBW_PACKED_ITEM>;
static_assert(LBW_PACKED_ITEM == PK_ITEM, "the kernels' item size");

}  // namespace

extern "C" {

int lbw_head_norm_rope(const lbw_head_norm_rope_params* p, void* stream) {
  HeadNormArgs a;
  LBW_TRY(fill_head_norm(p, &a));
  // (a wave per token, where tokens are few up to 32767 in all; the gradient's grid does not grow with them)
  if (p->tokens > HN_WAVES * kMaxWorkgroups)
    return fail(LBW_ERR_UNSUPPORTED, "tokens %d above %lld", p->tokens, (long long)(HN_WAVES * kMaxWorkgroups));
  LBW_TRY(check_rows("q_out", p->q_out, p->tokens, p->q_out_stride_l, p->q_out_stride_h));
  LBW_TRY(check_rows("k_out", p->k_out, p->tokens, p->k_out_stride_l, p->k_out_stride_h));
  LBW_TRY(check_head_strides("q_out", p->q_out_stride_h));
  LBW_TRY(check_head_strides("k_out", p->k_out_stride_h));
  a.qo = {static_cast<uint16_t*>(p->q_out), p->q_out_stride_l, p->q_out_stride_h};
  a.ko = {static_cast<uint16_t*>(p->k_out), p->k_out_stride_l, p->k_out_stride_h};
  if (p->v != nullptr) {
    LBW_TRY(check_rows("v", p->v, p->tokens, p->v_stride_l, p->v_stride_h));
    LBW_TRY(check_rows("v_out", p->v_out, p->tokens, p->v_out_stride_l, p->v_out_stride_h));
    LBW_TRY(check_head_strides("v", p->v_stride_h));
    LBW_TRY(check_head_strides("v_out", p->v_out_stride_h));
    a.v = {static_cast<const uint16_t*>(p->v), p->v_stride_l, p->v_stride_h};
    a.vo = {static_cast<uint16_t*>(p->v_out), p->v_out_stride_l, p->v_out_stride_h};
  }
  if (p->rows != nullptr) {
    if (p->row_count < 0 || !mult8(p->k_out_stride_b) || p->k_out_stride_b < 0 ||
        (p->v != nullptr && (!mult8(p->v_out_stride_b) || p->v_out_stride_b < 0)))
      return fail(LBW_ERR_INVALID, "rows: row_count %d, sequence strides must be multiples of 8",
                  p->row_count);
    a.rows = p->rows;
    a.cap = p->row_count;
    a.kosb = p->k_out_stride_b;
    a.vosb = p->v_out_stride_b;
  }
  if (p->tokens == 0) return LBW_OK;
  const hipError_t e = launch_head_norm(a, p->head_dim, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "head_norm_rope launch");
}

size_t lbw_head_norm_rope_bwd_workspace_size(const lbw_head_norm_rope_params* p) {
  if (p == nullptr || p->tokens <= 0 || p->head_dim <= 0) return 0;
  return (size_t)head_norm_bwd_workgroups(p->tokens, num_cus()) * p->head_dim * sizeof(float);
}

int lbw_head_norm_rope_bwd(const lbw_head_norm_rope_params* p, const lbw_head_norm_rope_grads* g,
                           void* workspace, size_t workspace_bytes, void* stream) {
  HeadNormArgs a;
  LBW_TRY(fill_head_norm(p, &a));
  if (g == nullptr) return fail(LBW_ERR_INVALID, "grads is NULL");
  LBW_TRY(check_rows("dq_out", g->dq_out, p->tokens, g->dq_out_stride_l, g->dq_out_stride_h));
  LBW_TRY(check_rows("dk_out", g->dk_out, p->tokens, g->dk_out_stride_l, g->dk_out_stride_h));
  LBW_TRY(check_rows("dq", g->dq, p->tokens, g->dq_stride_l, g->dq_stride_h));
  LBW_TRY(check_rows("dk", g->dk, p->tokens, g->dk_stride_l, g->dk_stride_h));
  LBW_TRY(check_head_strides("dq_out", g->dq_out_stride_h));
  LBW_TRY(check_head_strides("dk_out", g->dk_out_stride_h));
  LBW_TRY(check_head_strides("dq", g->dq_stride_h));
  LBW_TRY(check_head_strides("dk", g->dk_stride_h));
  const size_t need = lbw_head_norm_rope_bwd_workspace_size(p);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
    return fail(LBW_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need,
                workspace_bytes);
  a.dqo = {static_cast<const uint16_t*>(g->dq_out), g->dq_out_stride_l, g->dq_out_stride_h};
  a.dko = {static_cast<const uint16_t*>(g->dk_out), g->dk_out_stride_l, g->dk_out_stride_h};
  a.qo = {static_cast<uint16_t*>(g->dq), g->dq_stride_l, g->dq_stride_h};
  a.ko = {static_cast<uint16_t*>(g->dk), g->dk_stride_l, g->dk_stride_h};
  a.dwq = g->dwq;
  a.dwk = g->dwk;
  a.part = static_cast<float*>(workspace);
  a.nwg = head_norm_bwd_workgroups(p->tokens, num_cus());
  // (no tokens: the sum over no partial rows gives zero weight gradients)
  const hipError_t e = launch_head_norm_bwd(a, p->head_dim, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "head_norm_rope_bwd launch");
}

int lbw_attention_packed_plan(int32_t n_seqs, const int32_t* q_lens, const int32_t* k_lens,
                              int32_t causal, int32_t* q_items, int64_t q_items_cap,
                              int32_t* k_items, int64_t k_items_cap, lbw_packed_plan_info* info) {
  if (n_seqs < 0 || (n_seqs > 0 && (q_lens == nullptr || k_lens == nullptr)))
    return fail(LBW_ERR_INVALID, "n_seqs %d needs q_lens and k_lens", n_seqs);
  if (info == nullptr) return fail(LBW_ERR_INVALID, "info must not be NULL");
  int64_t tq = 0, tk = 0, nq = 0, nk = 0;
  for (int32_t s = 0; s < n_seqs; ++s) {
    if (q_lens[s] < 0 || k_lens[s] < 0)
      return fail(LBW_ERR_INVALID, "sequence %d: negative length", s);
    tq += q_lens[s];
    tk += k_lens[s];
    nq += (q_lens[s] + (int64_t)PK_BLOCK - 1) / PK_BLOCK;
    nk += (k_lens[s] + (int64_t)PK_BLOCK - 1) / PK_BLOCK;
  }
  if (tq > kMaxTokens || tk > kMaxTokens)
    return fail(LBW_ERR_UNSUPPORTED, "%lld query and %lld key rows: at most 2^31 - 256", (long long)tq,
                (long long)tk);
  memset(info, 0, sizeof(*info));
  info->n_q_items = nq;
  info->n_k_items = nk;
  for (int32_t s = 0; s < n_seqs; ++s) {
    const int64_t lq = q_lens[s], lk = k_lens[s], shift = causal ? lk - lq : lk;
    for (int64_t i = 0; i < lq; i += PK_BLOCK) {
      const int64_t seen = std::clamp<int64_t>(std::min<int64_t>(i + PK_BLOCK, lq) + shift, 0, lk);
      const int64_t t = (seen + 63) / 64;
      info->q_tiles += t;
      info->q_tiles_max = std::max(info->q_tiles_max, t);
    }
    for (int64_t j = 0; j < lk; j += PK_BLOCK) {
      const int64_t first = std::clamp<int64_t>(j - shift, 0, lq);
      const int64_t t = first < lq ? (lq + 63) / 64 - first / 64 : 0;
      info->k_tiles += t;
      info->k_tiles_max = std::max(info->k_tiles_max, t);
    }
  }
  if (q_items == nullptr && k_items == nullptr) return LBW_OK;
  if ((nq > 0 && q_items == nullptr) || (nk > 0 && k_items == nullptr) || q_items_cap < nq ||
      k_items_cap < nk)
    return fail(LBW_ERR_INVALID, "room for %lld and %lld items needed", (long long)nq, (long long)nk);
  try {
    std::vector<Item> qi, ki;
    qi.reserve(nq);
    ki.reserve(nk);
    int32_t q0 = 0, k0 = 0;
    for (int32_t s = 0; s < n_seqs; ++s) {
      const int32_t lq = q_lens[s], lk = k_lens[s];
      // full attention: a shift past every key
      const int32_t shift = causal ? lk - lq : lk;
      for (int64_t i = 0; i < lq; i += PK_BLOCK) {
        const int64_t rows = std::min<int64_t>(PK_BLOCK, lq - i);
        const int64_t seen = std::clamp<int64_t>(i + rows + shift, 0, lk);
        qi.push_back({q0 + (int32_t)i, (int32_t)rows, (int32_t)i, k0, lk, (int32_t)seen, shift, 0});
      }
      for (int64_t j = 0; j < lk; j += PK_BLOCK) {
        const int64_t rows = std::min<int64_t>(PK_BLOCK, lk - j);
        const int64_t first = std::clamp<int64_t>(j - shift, 0, lq);
        ki.push_back({k0 + (int32_t)j, (int32_t)rows, (int32_t)j, q0, lq, (int32_t)first, shift, 0});
      }
      q0 += lq;
      k0 += lk;
    }
    std::stable_sort(qi.begin(), qi.end(), [](const Item& x, const Item& y) { return x[5] > y[5]; });
    std::stable_sort(ki.begin(), ki.end(), [](const Item& x, const Item& y) {
      return (int64_t)x[4] - x[5] > (int64_t)y[4] - y[5];
    });
    if (nq > 0) memcpy(q_items, qi.data(), qi.size() * sizeof(Item));
    if (nk > 0) memcpy(k_items, ki.data(), ki.size() * sizeof(Item));
  } catch (const std::bad_alloc&) {
    return fail(LBW_ERR_INVALID, "no memory for %lld items", (long long)(nq + nk));
  }
  return LBW_OK;
}

size_t lbw_attention_packed_workspace_size(const lbw_packed_params* p) {
  return sane(p) ? part_bytes(split_q(p), p->q_heads, PK_PART_FWD) : 0;
}

int lbw_attention_packed_fwd(const lbw_packed_params* p, void* workspace, size_t workspace_bytes,
                             void* stream) {
  PackedArgs a;
  LBW_TRY(fill_packed(p, &a));
  if (a.n_q_items == 0) return LBW_OK;
  const PackedSplit s = split_q(p);
  LBW_TRY(check_grid(s, a.n_q_items, a.Hq, kMaxWorkgroups));
  const size_t need = part_bytes(s, p->q_heads, PK_PART_FWD);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
    return fail(LBW_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need,
                workspace_bytes);
  set_split(&a, s, workspace);
  const hipError_t e = launch_packed_fwd(a, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "packed attention launch");
}

// -delta and -lse / scale, then the partial results of dQ and, after them, of dK and dV in the same place
size_t lbw_attention_packed_bwd_workspace_size(const lbw_packed_params* p) {
  if (!sane(p)) return 0;
  return stat_bytes(p) + std::max(part_bytes(split_q(p), p->q_heads, PK_PART_DQ),
                                  part_bytes(split_k(p), p->k_heads, PK_PART_DKV));
}

int lbw_attention_packed_bwd(const lbw_packed_params* p, const lbw_packed_grads* g,
                             void* workspace, size_t workspace_bytes, void* stream) {
  PackedArgs a;
  LBW_TRY(fill_packed(p, &a));
  if (g == nullptr) return fail(LBW_ERR_INVALID, "grads is NULL");
  if (p->n_k_items < 0 || (p->n_k_items > 0 && p->k_items == nullptr))
    return fail(LBW_ERR_INVALID, "k_items missing");
  LBW_TRY(check_grid(split_q(p), p->n_q_items, p->q_heads, kMaxWorkgroups));
  LBW_TRY(check_grid(split_k(p), p->n_k_items, p->k_heads, kMaxWorkgroups / 2));
  if (p->q_tokens > 0 && p->lse == nullptr) return fail(LBW_ERR_INVALID, "lse missing");
  LBW_TRY(check_rows("dout", g->dout, p->q_tokens, g->dout_stride_l, g->dout_stride_h, true));
  LBW_TRY(check_rows("dq", g->dq, p->q_tokens, g->dq_stride_l, g->dq_stride_h));
  LBW_TRY(check_rows("dk", g->dk, p->k_tokens, g->dk_stride_l, g->dk_stride_h));
  LBW_TRY(check_rows("dv", g->dv, p->k_tokens, g->dv_stride_l, g->dv_stride_h));
  const size_t need = lbw_attention_packed_bwd_workspace_size(p);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
    return fail(LBW_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need,
                workspace_bytes);
  a.o = {static_cast<const uint16_t*>(p->out), p->out_stride_l, p->out_stride_h};
  a.dout = {static_cast<const uint16_t*>(g->dout), g->dout_stride_l, g->dout_stride_h};
  a.ndelta = static_cast<float*>(workspace);
  a.nlse = a.ndelta + (size_t)p->q_heads * (size_t)p->q_tokens;
  a.dq = {static_cast<uint16_t*>(g->dq), g->dq_stride_l, g->dq_stride_h};
  a.dk = {static_cast<uint16_t*>(g->dk), g->dk_stride_l, g->dk_stride_h};
  a.dv = {static_cast<uint16_t*>(g->dv), g->dv_stride_l, g->dv_stride_h};
  void* const part = static_cast<char*>(workspace) + stat_bytes(p);
  if (a.n_q_items > 0) {
    set_split(&a, split_q(p), part);
    const hipError_t e = launch_packed_dq(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "packed attention dQ launch");
  }
  if (a.n_k_items > 0) {
    const PackedSplit s = split_k(p);
    set_split(&a, s, part);
    a.halves = halves_k(p, s);
    const hipError_t e = launch_packed_dkv(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "packed attention dK/dV launch");
  }
  return LBW_OK;
}

size_t lbw_attention_decode_workspace_size(const lbw_decode_params* p) {
  if (check_decode(p) != LBW_OK || p->batch == 0) return 0;
  return decode_bytes(p, pieces_for(p));
}

int lbw_attention_decode(const lbw_decode_params* p, void* workspace, size_t workspace_bytes,
                         void* stream) {
  LBW_TRY(check_decode(p));
  const int64_t B = p->batch;
  LBW_TRY(check_rows("q", p->q, B, p->q_stride_b, p->q_stride_h));
  LBW_TRY(check_rows("out", p->out, B, p->out_stride_b, p->out_stride_h));
  LBW_TRY(check_rows("k", p->k, B * p->capacity, p->k_stride_l, p->k_stride_h, true));
  LBW_TRY(check_rows("v", p->v, B * p->capacity, p->v_stride_l, p->v_stride_h, true));
  if (!mult8(p->k_stride_b) || !mult8(p->v_stride_b) || p->k_stride_b < 0 || p->v_stride_b < 0)
    return fail(LBW_ERR_INVALID, "cache batch strides must be multiples of 8 elements");
  if (B > 0 && p->lens == nullptr) return fail(LBW_ERR_INVALID, "lens missing");
  DecodeArgs a;
  memset(&a, 0, sizeof(a));
  LBW_TRY(check_scale(p->softmax_scale, p->head_dim, &a.scale));
  if (B == 0) return LBW_OK;
  a.pieces = pieces_for(p);
  const size_t need = decode_bytes(p, a.pieces);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
    return fail(LBW_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need,
                workspace_bytes);
  a.q = {static_cast<const uint16_t*>(p->q), p->q_stride_b, p->q_stride_h};
  a.k = static_cast<const uint16_t*>(p->k);
  a.v = static_cast<const uint16_t*>(p->v);
  a.ksb = p->k_stride_b; a.ksl = p->k_stride_l; a.ksh = p->k_stride_h;
  a.vsb = p->v_stride_b; a.vsl = p->v_stride_l; a.vsh = p->v_stride_h;
  a.lens = p->lens;
  a.out = {static_cast<uint16_t*>(p->out), p->out_stride_b, p->out_stride_h};
  a.B = p->batch; a.Hq = p->q_heads; a.Hk = p->k_heads; a.S = (int)p->capacity;
  a.scale_log2 = (float)((double)a.scale * kLog2e);
  a.part = static_cast<float*>(workspace);
  const hipError_t e = launch_decode(a, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LBW_OK : hip_fail(e, "single-token attention launch");
}

}  // extern "C"
