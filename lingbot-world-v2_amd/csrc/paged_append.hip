// New tokens into a paged cache (gfx950): q and k normalised per head (or not) and turned by their positions, k and
// v put into their rows of the pages, and the smallest and largest value of each key component of a page kept up.
//
//   row r of token t: lens[b] + t - starts[b] (starts null: b = t, r = lens[t]); page table[b][r / P], row r % P.
//   y = x [rsqrt(mean_d x^2 + eps) w]; pair (a, b) of y turned by its angle, times `scale`; one rounding to bf16.
//   bounds[page] = (min, max) over the page's rows so far, of the rounded values: exact, so their order is free.
//
// Bound by memory: every value is read once and written once. As in the per-head norm a wave keeps a token, its
// angles in registers, and walks its heads. 4680 + 3600 + 1561 tokens x 40/8 heads of 128, normed, 54 us (5.2 TB/s; a
// large copy reaches 4.9), their pages' bounds 8 us; one token 4.3 us, most of it the launch.

#include "head_rows.h"
#include "paged.h"

namespace lbw {
namespace {

constexpr int AP_WAVES = 4;
constexpr int EDGE_WAVES = 8;  // of the bounds kernel

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

// The smaller and the larger of two values, NaN if one of them is.
__device__ __forceinline__ float min_nan(float x, float y) { return __builtin_elementwise_minimum(x, y); }
__device__ __forceinline__ float max_nan(float x, float y) { return __builtin_elementwise_maximum(x, y); }

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
template <int LPH, bool INTER>
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
      *reinterpret_cast<u32x4*>(dst + (int64_t)ch * HPW * dsh + dof) = out;
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

template <int LPH>
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
      if (ch * HPW + hsub < heads) *reinterpret_cast<u32x4*>(dst + (int64_t)ch * HPW * dsh + dof) = x[u];
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

template <int LPH, bool INTER>
__global__ void __launch_bounds__(AP_WAVES * 64) append_kernel(const AppendArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * AP_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  turn_rows<LPH, INTER>(a, a.q.p + t * a.q.sl, a.q.sh, a.qo.p + t * a.qo.sl, a.qo.sh, a.Hq, part, a.parts, e0, hsub,
                        a.wq, a.q_scale, rot, nullptr, false);
  if (w.page < 0) return;
  const int64_t in = w.row & ((1 << a.pt.shift) - 1);
  // one new token per sequence: its page's bounds are this wave's
  uint16_t* const bounds =
      a.bounds != nullptr && a.starts == nullptr ? a.bounds + (int64_t)w.page * a.Hk * 2 * D : nullptr;
  turn_rows<LPH, INTER>(a, a.k.p + t * a.k.sl, a.k.sh, a.kp.p + w.page * a.kp.sp + in * a.kp.sl, a.kp.sh, a.Hk,
                        first(cq), a.parts, e0, hsub, a.wk, a.k_scale, rot, bounds, in == 0);
  copy_rows<LPH>(a.v.p + t * a.v.sl, a.v.sh, a.vp.p + w.page * a.vp.sp + in * a.vp.sl, a.vp.sh, a.Hk,
                 first(cq + ck), a.parts, e0, hsub);
}

// Bounds of the pages that several tokens were put into: blockIdx.x counts blocks of a.run_block tokens, blockIdx.y
// chunks of heads. The workgroup whose block holds a page's first new token reads the page's new keys back (from
// cache: they were written just before), its waves in turn, and joins them with the old bounds where the page was
// begun before: every page has one owner, no atomics. (One kernel, in which the workgroup that makes a page's bounds
// turns its keys: 4680 + 3600 + 1561 tokens x 40/8 heads 69 to 90 us against 54 + 8, as a page's tokens follow one
// another.)
template <int LPH>
__global__ void __launch_bounds__(EDGE_WAVES * 64) append_bounds_kernel(const AppendArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH, U = 8;
  __shared__ u32x4 red[2][EDGE_WAVES][64];  // (bf16: what was rounded once stays)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = 8 * (lane % LPH), head = (int)blockIdx.y * HPW + lane / LPH;
  const int hh = head < a.Hk ? head : a.Hk - 1;  // (lanes past the last head do its work again and write nothing)
  const int64_t t0 = (int64_t)blockIdx.x * a.run_block;
  const int t1 = (int)(t0 + a.run_block < a.T ? t0 + a.run_block : a.T);
  const int mask = (1 << a.pt.shift) - 1;
  for (int t = (int)t0; t < t1;) {
    const Place w = place_of(a, t, lane);
    if (w.b < 0) {
      ++t;
      continue;
    }
    const int in = (int)(w.row & mask);
    const int n = w.end - t < mask + 1 - in ? w.end - t : mask + 1 - in;  // this page's tokens from t on
    if (w.page < 0 || (in != 0 && t != w.start)) {  // nowhere, or not its first new token
      t += n;
      continue;
    }
    const uint16_t* const rows = a.kp.p + w.page * a.kp.sp + in * a.kp.sl + hh * a.kp.sh + e0;
    uint16_t* const edge = a.bounds + ((int64_t)w.page * a.Hk + hh) * 2 * D + (wave & 1) * D + e0;
    const u32x4 before = load16(edge);
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = INFINITY;
      hi[j] = -INFINITY;
    }
    for (int r = wave; r < n; r += EDGE_WAVES * U) {
      u32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (past the end: the last row once more)
        const int rr = r + u * EDGE_WAVES < n ? r + u * EDGE_WAVES : n - 1;
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
    __syncthreads();  // the last page's results are read
    red[0][wave][lane] = pack8(lo);
    red[1][wave][lane] = pack8(hi);
    __syncthreads();
    if (wave < 2 && head < a.Hk) {  // one wave for the smallest values, one for the largest
      float m[8], y[8];
      unpack8(in != 0 ? before : red[wave][0][lane], m);
#pragma unroll
      for (int x = 0; x < EDGE_WAVES; ++x) {
        unpack8(red[wave][x][lane], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = wave == 0 ? min_nan(m[j], y[j]) : max_nan(m[j], y[j]);
      }
      *reinterpret_cast<u32x4*>(edge) = pack8(m);
    }
    t += n;
  }
}

template <int LPH>
hipError_t run(AppendArgs a, hipStream_t stream) {
  constexpr int HPW = 64 / LPH;
  const int64_t waves = (int64_t)a.T * a.parts;
  const dim3 grid((uint32_t)((waves + AP_WAVES - 1) / AP_WAVES)), block(AP_WAVES * 64);
  if (a.inter) hipLaunchKernelGGL((append_kernel<LPH, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((append_kernel<LPH, false>), grid, block, 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.bounds == nullptr || a.starts == nullptr) return e;
  // as many tokens as a page has, so that a workgroup finds one page to look after, or fewer where sequences are
  // shorter or workgroups few (a page takes its workgroup some microseconds, most of them waiting)
  a.run_block = 1;
  while (a.run_block < (1 << a.pt.shift) && (int64_t)2 * a.run_block * a.B <= a.T && a.T / a.run_block > 512)
    a.run_block *= 2;
  const dim3 runs((a.T + a.run_block - 1) / a.run_block, (a.Hk + HPW - 1) / HPW);
  hipLaunchKernelGGL(append_bounds_kernel<LPH>, runs, dim3(EDGE_WAVES * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_append(const AppendArgs& args, int D, hipStream_t stream) {
  AppendArgs a = args;
  // a token's heads are shared by several waves while the tokens alone do not fill the chip
  const int nch = (a.Hq + 2 * a.Hk + 512 / D - 1) / (512 / D);
  a.parts = 1;
  while (a.parts < nch && (int64_t)a.T * a.parts < 16384) a.parts *= 2;
  switch (D) {
    case 32: return run<4>(a, stream);
    case 64: return run<8>(a, stream);
    case 128: return run<16>(a, stream);
    default: return run<32>(a, stream);
  }
}

}  // namespace lbw
