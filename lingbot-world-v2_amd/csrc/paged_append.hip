// New tokens into a paged cache (gfx950): q and k normalised per head (or not) and turned by their positions, k and
// v put into their rows of the pages, and the smallest and largest value of each key component of a page kept up.
//
//   row r of token t: lens[b] + t - starts[b] (starts null: b = t, r = lens[t]); page table[b][r / P], row r % P.
//   y = x [rsqrt(mean_d x^2 + eps) w]; pair (a, b) of y turned by its angle, times `scale`; one rounding to bf16.
//   bounds[page] = (min, max) over the page's rows so far, of the rounded values: exact, so their order is free.
//
// Bound by memory: every value is read once and written once. As in the per-head norm a wave keeps a token, its
// angles in registers, and walks its heads. Several tokens for one page: the keys are turned by the workgroup that
// makes the page's bounds, beside the tokens' q and v. 4680 + 3600 + 1561 tokens x 40/8 heads of 128, normed, pages of 64,
// from memory 62 us (4.6 TB/s; a large copy reaches 4.9), inputs in the last cache 46; one token 4.4 us, most of it the launch.

#include <algorithm>

#include "capi_util.h"
#include "head_rows.h"
#include "paged.h"

namespace lbw {
namespace {

constexpr int AP_WAVES = 4;
constexpr int KEY_HEADS = 2;   // heads of a workgroup that looks after a page's keys, at most
constexpr int EDGE_WAVES = 8;  // of the bounds kernel
// Pages that can get up to so many new tokens get their keys and bounds in the kernel of the tokens' q and v, others, whose
// tokens would follow one another too long, their bounds by a second kernel. Two kernels / one, x 40/8 heads, pages of 64: 100 tokens
// 12.5 / 10.1 us, 500 12.5 / 11.4, 2000 17.7 / 14.8, 4680 35.6 / 35.0, 9841 67.5 / 60.1; of 128 11.9 / 13.2, 12.9 / 17.3, 18.9 / 20.1,
// 36.6 / 38.7, 67.0 / 62.3; of 256 11.8 / 13.2, 14.4 / 29.4, 20.5 / 31.8, 37.6 / 48.7, 67.6 / 73.2.
constexpr int FUSED_PAGE = 64;

// Where a token goes: its sequence (-1: none), row and page (-1: nowhere).
struct Place {
  int b;
  int64_t row;
  int page;
  int start, end;  // the sequence's tokens
};
__device__ __forceinline__ Place place_of(const AppendArgs& a, int t, int lane) {
  Place w = {t, 0, -1, t, t + 1};
  int len;
  if (a.starts == nullptr) {
    len = __builtin_amdgcn_readfirstlane(a.lens[t]);
  } else {
    // the last sequence that starts at or before the token: 64 starts at a time, and at the end all that is wanted
    // of the sequence in one go
    int base = 0, n = a.B;
    while (n > 64) {
      const int step = (n + 63) >> 6, off = lane * step;
      const uint64_t past = __ballot(off < n && a.starts[base + off] <= t);
      if (past == 0) break;
      const int c = (63 - __clzll((unsigned long long)past)) * step;
      base += c;
      n = n - c < step ? n - c : step;
    }
    int s = 0, e = 0, l = 0;
    const bool mine = lane < n;
    if (mine) {
      s = a.starts[base + lane];
      e = a.starts[base + lane + 1];
      l = a.lens[base + lane];
    }
    const uint64_t past = __ballot(mine && s <= t);
    const int c = past == 0 ? 0 : 63 - __clzll((unsigned long long)past);
    w.b = past == 0 ? -1 : base + c;
    w.start = __builtin_amdgcn_readlane(s, c);
    w.end = __builtin_amdgcn_readlane(e, c);
    w.end = w.end < a.T ? w.end : a.T;
    len = __builtin_amdgcn_readlane(l, c);
    if (t >= w.end) w.b = -1;  // behind the last sequence
    if (w.b < 0) return w;
  }
  w.row = (int64_t)len + ((int64_t)t - w.start);
  w.page = __builtin_amdgcn_readfirstlane(
      page_at(a.pt.p + (int64_t)w.b * a.pt.sb, a.pt.width, a.pt.shift, a.pt.pages, w.row));
  return w;
}

// A page's new tokens, of page `page`. Its owner is a workgroup: number `slot` of those that a.page_slots tells from one
// another by pages (first_owner), else by tokens. False: no page is here (or the sequence's table does not hold it).
struct Fresh : PageRun {
  int page;
};
__device__ __forceinline__ bool fresh_page(const AppendArgs& a, int64_t slot, int lane, Fresh& f) {
  const int shift = a.pt.shift;
  if (a.page_slots == 0) {
    const Place w = place_of(a, (int)slot, lane);
    if (w.b < 0 || w.page < 0) return false;
    f.page = w.page;
    return opened_run((int)slot, w.row, w.start, w.end, a.T, shift, f);
  }
  // the last sequence whose first slot is this one or before
  int base = 0, left = a.B;
  while (left > 64) {
    const int step = (left + 63) >> 6, off = lane * step;
    const uint64_t past = __ballot(off < left && first_owner(base + off, a.starts[base + off], shift) <= slot);
    if (past == 0) return false;
    const int c = (63 - __clzll((unsigned long long)past)) * step;
    base += c;
    left = left - c < step ? left - c : step;
  }
  int s = 0, e = 0, l = 0;
  const bool mine = lane < left;
  if (mine) {
    s = a.starts[base + lane];
    e = a.starts[base + lane + 1];
    l = a.lens[base + lane];
  }
  const uint64_t past = __ballot(mine && first_owner(base + lane, s, shift) <= slot);
  if (past == 0) return false;
  const int c = 63 - __clzll((unsigned long long)past), b = base + c;
  const int start = __builtin_amdgcn_readlane(s, c), stop = __builtin_amdgcn_readlane(e, c);
  if (!owned_run(start, stop, a.T, __builtin_amdgcn_readlane(l, c), shift, slot - first_owner(b, start, shift), f)) return false;
  f.page = __builtin_amdgcn_readfirstlane(
      page_at(a.pt.p + (int64_t)b * a.pt.sb, a.pt.width, shift, a.pt.pages, f.row));
  return f.page >= 0;
}

// The smaller and the larger of two values, NaN if one of them is.
__device__ __forceinline__ float min_nan(float x, float y) { return __builtin_elementwise_minimum(x, y); }
__device__ __forceinline__ float max_nan(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// A chunk of a row. PAST: past the caches, for prompts' rows in their pages, which the next call mostly does not read in
// full; q, and a decoded token's row, are read next. Prompts x 40/8 heads, inputs from memory, into the caches / past: 1000
// tokens 23.6 / 22.6 us, 2000 32.1 / 31.9, 4680 37.8 / 37.4, 9841 61.5 / 60.4 (inputs in the last cache 54.6 / 45); with q read
// by a copy behind it 28.3 / 27.5, 39.5 / 39.1, 51.3 / 50.7, 97.0 / 95.8 (q past the caches too: 26.9, 39.4, 52.4, 96.1). No
// bounds: 3500 tokens 29.4 / 24.4, 9841 61.7 / 59.7.
template <bool PAST>
__device__ __forceinline__ void put16(uint16_t* p, const u32x4& x) {
  if constexpr (PAST) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = x;
}

// Eight values of a head: normed (or not), turned, scaled, rounded.
template <int LPH, bool INTER>
__device__ __forceinline__ u32x4 turn_chunk(const AppendArgs& a, const u32x4& x, const float (&wt)[8], float scale,
                                            const Turn& rot) {
  float f[8], o[8];
  unpack8(x, f);
  float r = scale;
  if (a.norm) {
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
    r = rsqrtf(head_sum<LPH>(ss) * a.inv_d + a.eps) * scale;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= r * wt[j];
  turn<INTER, false>(rot, f, o);
  return pack8(o);
}

// Chunks first, first + step, .. of a token's heads; `bounds` (of the token's page, or null): the page's, started anew
// if `fresh`.
template <int LPH, bool INTER, bool PAST>
__device__ __forceinline__ void turn_rows(const AppendArgs& a, const uint16_t* src, int64_t ssh, uint16_t* dst,
                                          int64_t dsh, int heads, int first, int step, int e0, int hsub,
                                          const void* w, float scale, const Turn& rot, uint16_t* bounds, bool fresh) {
  constexpr int HPW = 64 / LPH, U = 4, D = 8 * LPH;
  const int nch = (heads + HPW - 1) / HPW;
  if (first >= nch) return;
  const uint32_t so = (uint32_t)(hsub * (int)ssh + e0), dof = (uint32_t)(hsub * (int)dsh + e0);
  float wt[8];
  load_weights(w, a.w32, e0, wt);
  for (int it = first; it < nch; it += U * step) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      x[u] = u32x4{0u, 0u, 0u, 0u};
      if (ch * HPW + hsub < heads) x[u] = load16(src + (int64_t)ch * HPW * ssh + so);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      if (ch >= nch) break;
      const u32x4 out = turn_chunk<LPH, INTER>(a, x[u], wt, scale, rot);
      if (ch * HPW + hsub >= heads) continue;
      put16<PAST>(dst + (int64_t)ch * HPW * dsh + dof, out);
      if (bounds == nullptr) continue;
      uint16_t* const lo = bounds + (int64_t)(ch * HPW + hsub) * 2 * D + e0;
      u32x4 l = out, h = out;
      if (!fresh) {
        float v[8], m[8];
        unpack8(out, v);
        unpack8(load16(lo), m);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = min_nan(m[j], v[j]);
        l = pack8(m);
        unpack8(load16(lo + D), m);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = max_nan(m[j], v[j]);
        h = pack8(m);
      }
      *reinterpret_cast<u32x4*>(lo) = l;
      *reinterpret_cast<u32x4*>(lo + D) = h;
    }
  }
}

template <int LPH, bool PAST>
__device__ __forceinline__ void copy_rows(const uint16_t* src, int64_t ssh, uint16_t* dst, int64_t dsh, int heads,
                                          int first, int step, int e0, int hsub) {
  constexpr int HPW = 64 / LPH, U = 4;
  const int nch = (heads + HPW - 1) / HPW;
  const uint32_t so = (uint32_t)(hsub * (int)ssh + e0), dof = (uint32_t)(hsub * (int)dsh + e0);
  for (int it = first; it < nch; it += U * step) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      if (ch * HPW + hsub < heads) x[u] = load16(src + (int64_t)ch * HPW * ssh + so);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      if (ch * HPW + hsub < heads) put16<PAST>(dst + (int64_t)ch * HPW * dsh + dof, x[u]);
    }
  }
}

// The rotation of token t, at `row` of its sequence.
template <bool INTER>
__device__ __forceinline__ void load_rotation(const AppendArgs& a, int t, int64_t row, int e0, int lane, Turn& rot) {
  if (a.pos != nullptr) {
    load_turn<INTER>(a, t, e0, lane, rot);
  } else {
    // (a row past 31 bits is outside every table)
    const int p = row >= 0 && row < a.P ? (int)row : -1;
    load_turn_at<INTER>(a, p, p, p, p, e0, lane, rot);
  }
}

// The page's new keys, turned and put there, heads h0 .., and its bounds, made of them and, where the page was begun
// before, the old ones: every page has one owner, no atomics. A wave takes 64 / LPH tokens at a time, a head after the
// other, so that a token's angles are read once; the tokens' smallest and largest values meet by shuffles, the waves'
// in LDS.
template <int LPH, bool INTER>
__device__ __forceinline__ void append_page(const AppendArgs& a, const Fresh& f, int chunk, int lane, int wave) {
  constexpr int TPW = 64 / LPH, D = 8 * LPH, KH = KEY_HEADS;
  __shared__ u32x4 red[AP_WAVES][KH][2][LPH];  // (bf16: what was rounded once stays)
  const int e0 = 8 * (lane % LPH), sub = lane / LPH, h0 = chunk * a.page_heads;
  const int h1 = h0 + a.page_heads < a.Hk ? h0 + a.page_heads : a.Hk;  // heads h0 .. h1 - 1
  float wt[8];
  load_weights(a.wk, a.w32, e0, wt);
  const int turns = (f.n + TPW - 1) / TPW;
  for (int g = wave; g < turns; g += AP_WAVES) {
    const int mine = g * TPW + sub, tok = mine < f.n ? mine : f.n - 1;  // (past the end: the last one once more)
    u32x4 x[KH];
    const uint16_t* const src = a.k.p + (int64_t)(f.t + tok) * a.k.sl + e0;
#pragma unroll
    for (int i = 0; i < KH; ++i) x[i] = load16(src + (h0 + i < h1 ? h0 + i : h0) * a.k.sh);
    Turn rot;
    load_rotation<INTER>(a, f.t + tok, f.row + tok, e0, lane, rot);
    uint16_t* const dst = a.kp.p + f.page * a.kp.sp + (f.in + tok) * a.kp.sl + e0;
#pragma unroll
    for (int i = 0; i < KH; ++i) {
      if (h0 + i >= h1) break;
      const u32x4 out = turn_chunk<LPH, INTER>(a, x[i], wt, a.k_scale, rot);
      if (mine < f.n) put16<true>(dst + (h0 + i) * a.kp.sh, out);
      float lo[8], hi[8], y[8];
      unpack8(out, lo);
      unpack8(out, hi);
      u32x4 pl = out, ph = out;
#pragma unroll
      for (int o = LPH; o < 64; o <<= 1) {
        u32x4 ql, qh;
#pragma unroll
        for (int e = 0; e < 4; ++e) ql[e] = __shfl_xor(pl[e], o);
        qh = ql;
        if (o > LPH) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qh[e] = __shfl_xor(ph[e], o);
        }
        unpack8(ql, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = min_nan(lo[j], y[j]);
        unpack8(qh, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) hi[j] = max_nan(hi[j], y[j]);
        pl = pack8(lo);
        ph = pack8(hi);
      }
      if (lane < LPH) {
        if (g != wave) {
          unpack8(red[wave][i][0][lane], y);
#pragma unroll
          for (int j = 0; j < 8; ++j) lo[j] = min_nan(lo[j], y[j]);
          unpack8(red[wave][i][1][lane], y);
#pragma unroll
          for (int j = 0; j < 8; ++j) hi[j] = max_nan(hi[j], y[j]);
        }
        red[wave][i][0][lane] = pack8(lo);
        red[wave][i][1][lane] = pack8(hi);
      }
    }
  }
  __syncthreads();
  const int used = turns < AP_WAVES ? turns : AP_WAVES;
  for (int x = threadIdx.x; x < KH * 2 * LPH; x += AP_WAVES * 64) {
    const int c = x % LPH, edge = x / LPH % 2, i = x / (2 * LPH);
    if (h0 + i >= h1) break;
    uint16_t* const p = a.bounds + (((int64_t)f.page * a.Hk + h0 + i) * 2 + edge) * D + 8 * c;
    float m[8], y[8];
    unpack8(f.in != 0 ? load16(p) : red[0][i][edge][c], m);
    for (int v = 0; v < used; ++v) {
      unpack8(red[v][i][edge][c], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = edge == 0 ? min_nan(m[j], y[j]) : max_nan(m[j], y[j]);
    }
    *reinterpret_cast<u32x4*>(p) = pack8(m);
  }
}

// One token of each sequence, prompts' rows, or (PAGES) the first a.page_wgs workgroups look after the new keys of whole
// pages, the others after the tokens' q and v.
enum Keys { TOKEN, ROWS, PAGES };
template <int LPH, bool INTER, Keys KEYS>
__global__ void __launch_bounds__(AP_WAVES * 64) append_kernel(const AppendArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t wg = blockIdx.x;
  if constexpr (KEYS == PAGES) {
    if (wg < (uint32_t)a.page_wgs) {
      const uint32_t chunks = (uint32_t)((a.Hk + a.page_heads - 1) / a.page_heads);
      Fresh f;
      if (fresh_page(a, wg / chunks, lane, f)) append_page<LPH, INTER>(a, f, wg % chunks, lane, wave);
      return;
    }
    wg -= a.page_wgs;
  }
  const int64_t id = (int64_t)wg * AP_WAVES + wave;
  const int64_t tt = id / a.parts;
  if (tt >= a.T) return;
  const int t = (int)tt, part = (int)(id % a.parts);
  const int e0 = 8 * (lane % LPH), hsub = lane / LPH;
  const Place w = place_of(a, t, lane);
  if (w.b < 0) return;  // a row behind the last sequence: left as it was
  Turn rot;
  load_rotation<INTER>(a, t, w.row, e0, lane, rot);
  // the token's chunks, q's, k's, v's, in turn to the waves that share it
  const int cq = (a.Hq + HPW - 1) / HPW, ck = (a.Hk + HPW - 1) / HPW;
  auto first = [&](int before) {
    const int x = (part - before) % a.parts;
    return x < 0 ? x + a.parts : x;
  };
  turn_rows<LPH, INTER, false>(a, a.q.p + t * a.q.sl, a.q.sh, a.qo.p + t * a.qo.sl, a.qo.sh, a.Hq, part, a.parts, e0,
                               hsub, a.wq, a.q_scale, rot, nullptr, false);
  if (w.page < 0) return;
  const int64_t in = w.row & ((1 << a.pt.shift) - 1);
  const uint16_t *const k = a.k.p + t * a.k.sl, *const v = a.v.p + t * a.v.sl;
  uint16_t *const kp = a.kp.p + w.page * a.kp.sp + in * a.kp.sl, *const vp = a.vp.p + w.page * a.vp.sp + in * a.vp.sl;
  if constexpr (KEYS == TOKEN) {
    // one new token per sequence: its page's bounds are this wave's
    uint16_t* const bounds = a.bounds != nullptr ? a.bounds + (int64_t)w.page * a.Hk * 2 * D : nullptr;
    turn_rows<LPH, INTER, false>(a, k, a.k.sh, kp, a.kp.sh, a.Hk, first(cq), a.parts, e0, hsub, a.wk, a.k_scale, rot,
                                 bounds, in == 0);
  } else if constexpr (KEYS == ROWS) {
    if (a.bounds == nullptr) {
      turn_rows<LPH, INTER, true>(a, k, a.k.sh, kp, a.kp.sh, a.Hk, first(cq), a.parts, e0, hsub, a.wk, a.k_scale, rot,
                                  nullptr, false);
    } else {  // (the bounds kernel reads them)
      turn_rows<LPH, INTER, false>(a, k, a.k.sh, kp, a.kp.sh, a.Hk, first(cq), a.parts, e0, hsub, a.wk, a.k_scale, rot,
                                   nullptr, false);
    }
  }
  copy_rows<LPH, KEYS != TOKEN>(v, a.v.sh, vp, a.vp.sh, a.Hk, first(KEYS == PAGES ? cq : cq + ck), a.parts, e0, hsub);
}

// Bounds of the pages that several tokens were put into: a workgroup a page (blockIdx.x: fresh_page's slot) and chunk of
// heads (blockIdx.y) reads the page's new keys back (from cache: they were written just before), its waves in turn, and
// joins them with the old bounds where the page was begun before.
template <int LPH>
__global__ void __launch_bounds__(EDGE_WAVES * 64) append_bounds_kernel(const AppendArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH, U = 8;
  __shared__ u32x4 red[2][EDGE_WAVES][64];  // (bf16: what was rounded once stays)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = 8 * (lane % LPH), head = (int)blockIdx.y * HPW + lane / LPH;
  const int hh = head < a.Hk ? head : a.Hk - 1;  // (lanes past the last head do its work again and write nothing)
  Fresh w;
  if (!fresh_page(a, blockIdx.x, lane, w)) return;
  const uint16_t* const rows = a.kp.p + w.page * a.kp.sp + w.in * a.kp.sl + hh * a.kp.sh + e0;
  uint16_t* const edge = a.bounds + ((int64_t)w.page * a.Hk + hh) * 2 * D + (wave & 1) * D + e0;
  const u32x4 before = load16(edge);
  float lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo[j] = INFINITY;
    hi[j] = -INFINITY;
  }
  for (int r = wave; r < w.n; r += EDGE_WAVES * U) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the end: the last row once more)
      const int rr = r + u * EDGE_WAVES < w.n ? r + u * EDGE_WAVES : w.n - 1;
      x[u] = load16(rows + (int64_t)rr * a.kp.sl);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      unpack8(x[u], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = min_nan(lo[j], f[j]);
        hi[j] = max_nan(hi[j], f[j]);
      }
    }
  }
  red[0][wave][lane] = pack8(lo);
  red[1][wave][lane] = pack8(hi);
  __syncthreads();
  if (wave < 2 && head < a.Hk) {  // one wave for the smallest values, one for the largest
    float m[8], y[8];
    unpack8(w.in != 0 ? before : red[wave][0][lane], m);
#pragma unroll
    for (int x = 0; x < EDGE_WAVES; ++x) {
      unpack8(red[wave][x][lane], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = wave == 0 ? min_nan(m[j], y[j]) : max_nan(m[j], y[j]);
    }
    *reinterpret_cast<u32x4*>(edge) = pack8(m);
  }
}

template <int LPH, Keys KEYS>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
  const int64_t waves = (int64_t)a.T * a.parts;
  const dim3 grid((uint32_t)(a.page_wgs + (waves + AP_WAVES - 1) / AP_WAVES)), block(AP_WAVES * 64);
  if (a.inter) hipLaunchKernelGGL((append_kernel<LPH, true, KEYS>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((append_kernel<LPH, false, KEYS>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <int LPH>
hipError_t run(AppendArgs a, hipStream_t stream) {
  constexpr int HPW = 64 / LPH;
  a.page_wgs = 0;
  if (a.starts == nullptr) return launch<LPH, TOKEN>(a, stream);
  if (a.bounds == nullptr) return launch<LPH, ROWS>(a, stream);
  const int page = 1 << a.pt.shift;
  // a workgroup for every page that the sequences can touch, or every token where that is less (blocks of tokens searched
  // for pages, four times as many workgroups / half as many as CUs / a workgroup a page: 1000 tokens x 40/8 heads in pages of
  // 64 16.8 / 12.5 / 12.7 us, x 40/40 25.1 / 17.7 / 17.1, eight times 400 23.4 / 33.8 / 25.1, 400 + 4 x 40 + 3 x 4 x 12/12 in pages of 32
  // 12.4 / 18.7 / 10.8; 2000 x 40/40 in pages of 128, two kernels, 61.3 / 34.7 / 34.5)
  const int64_t slots = page_owners(a.T, a.B, a.pt.shift);
  a.page_slots = slots < a.T;
  const int owners = (int)std::min<int64_t>(slots, a.T);
  if (std::min(page, a.T) <= FUSED_PAGE) {
    // a head a workgroup, not two, while pages are few: two / one, in pages of 64, 500 tokens x 40/8 heads (32 workgroups of
    // two) 13.5 / 11.4 us, 2000 (128) 16.2 / 14.8, 2500 (160) 16.6 / 16.9, 3500 (220) 21.2 / 22.2, 2000 x 12/12 (192) 14.4 / 12.9
    const int64_t pages = (a.T >> a.pt.shift) + a.B;
    a.page_heads = pages * ((a.Hk + KEY_HEADS - 1) / KEY_HEADS) <= 3 * num_cus() / 4 ? 1 : KEY_HEADS;
    a.page_wgs = owners * ((a.Hk + a.page_heads - 1) / a.page_heads);
    return launch<LPH, PAGES>(a, stream);
  }
  const hipError_t e = launch<LPH, ROWS>(a, stream);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(append_bounds_kernel<LPH>, dim3(owners, (a.Hk + HPW - 1) / HPW), dim3(EDGE_WAVES * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_append(const AppendArgs& args, int D, hipStream_t stream) {
  AppendArgs a = args;
  // a token's heads are shared by several waves while the tokens alone do not fill the chip, up to 7000 waves: each of them
  // reads the token's place and angles (up to 16384 waves / up to 4096, 3000 tokens x 40/8 heads 31.8 / 23.0 us, 5000 x 12/12
  // 27.8 / 21.2, 16000 83 / 70; up to 8191 / 7000 / 5200, 1000 x 40/8 without bounds 11.4 / 9.5 / 9.4, 1500, from memory, 13.3 / 13.2
  // / 14.8, 2000 18.6 / 16.8 / 16.8, 3500 24.5 / 24.3 / 25.2)
  const int nch = (a.Hq + 2 * a.Hk + 512 / D - 1) / (512 / D);
  a.parts = 1;
  while (a.parts < nch && (int64_t)a.T * a.parts * 2 <= 7000) a.parts *= 2;
  switch (D) {
    case 32: return run<4>(a, stream);
    case 64: return run<8>(a, stream);
    case 128: return run<16>(a, stream);
    default: return run<32>(a, stream);
  }
}

}  // namespace lbw
