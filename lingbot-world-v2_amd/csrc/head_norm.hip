// RMSNorm of every query and key head and the rotation of its pairs, in one pass (gfx950), with
// its gradient.
//
//   y = x rsqrt(mean_d x^2 + eps) w;  pair (a, b) of y turned by its angle t, times `scale`:
//   (a cos t - b sin t, a sin t + b cos t); one rounding to bf16 at the end.
//   With g = scale R^T dy, r = rsqrt(mean x^2 + eps):
//   dw = sum over tokens and heads of g x r;  dx = r (g w - x r mean_d(g w x r)).
//
// Bound by memory: forward reads and writes each value once, the gradient reads two values and
// writes one. D / 8 lanes hold a head, 16 bytes each, so a wave covers 512 / D heads and the sums
// over a head are shuffles among its lanes. A wave keeps one token: its angles are read once into
// registers (cos and signed sin of the lane's eight values) and serve all its heads.

#include "common.h"
#include "packed.h"

namespace lbw {
namespace {

constexpr int HN_WAVES = 4;  // waves per workgroup

__device__ __forceinline__ void unpack8(const u32x4& v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(v[i]);
    x[2 * i + 1] = bf16_hi(v[i]);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return v;
}
__device__ __forceinline__ u32x4 load16(const uint16_t* p) { return *reinterpret_cast<const u32x4*>(p); }

// The lane's eight weights (1 without weights).
__device__ __forceinline__ void load_weights(const void* w, int w32, int e0, float (&x)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 1.0f;
  } else if (w32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = static_cast<const float*>(w)[e0 + j];
  } else {
    unpack8(load16(static_cast<const uint16_t*>(w) + e0), x);
  }
}

// Sum over the LPH lanes of a head, in every one of them.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Rotation of the lane's eight values e0 .. e0 + 7 of a head: value j becomes
// y[j] c[j] + partner[j] s[j], where its partner is the pair's other value.
struct Turn {
  float c[8], s[8];
  int lane;  // split halves: the lane that holds the partners (the own one: not rotated)
};

__device__ __forceinline__ void load_turn(const HeadNormArgs& a, int t, int e0, int lane, Turn& r) {
  const int h = a.npairs;
  // the axes' table rows; a position outside the table turns by NaN
  int64_t row[kMaxAxes];
#pragma unroll
  for (int x = 0; x < kMaxAxes; ++x) {
    const int p = x < a.naxes ? a.pos[t * a.pos_sl + x] : 0;
    row[x] = (p < 0 || p >= a.P) ? -1 : (int64_t)p * h;
  }
  const bool second = !a.inter && e0 >= h;
  const bool halves_rot = !a.inter && e0 < 2 * h;
  r.lane = halves_rot ? (second ? lane - h / 8 : lane + h / 8) : lane;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = a.inter ? (e0 + j) >> 1 : (second ? e0 + j - h : e0 + j);
    float c = 1.0f, s = 0.0f;
    if (i < h) {
      int64_t base = row[0];
      if (i >= a.ax_end[0]) base = row[1];
      if (i >= a.ax_end[1]) base = row[2];
      if (i >= a.ax_end[2]) base = row[3];
      float2 cs = {__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u)};
      if (base >= 0) cs = a.table[base + i];
      c = cs.x;
      s = (a.inter ? (j & 1) == 0 : !second) ? -cs.y : cs.y;
    }
    r.c[j] = c;
    r.s[j] = s;
  }
}

// y turned; back: by the negative angle.
template <bool BACK>
__device__ __forceinline__ void turn(const Turn& r, bool inter, const float (&y)[8], float (&o)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float p = inter ? y[j ^ 1] : __shfl(y[j], r.lane);
    o[j] = y[j] * r.c[j] + p * (BACK ? -r.s[j] : r.s[j]);
  }
}

template <int LPH>
__global__ void __launch_bounds__(HN_WAVES * 64) head_norm_kernel(const HeadNormArgs a) {
  constexpr int HPW = 64 / LPH;  // heads of one wave step
  constexpr int U = 4;           // steps in flight
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * HN_WAVES + (threadIdx.x >> 6);
  const int64_t tt = id / a.parts;
  if (tt >= a.T) return;
  const int t = (int)tt, part = (int)(id % a.parts);
  const int e0 = 8 * (lane % LPH), hsub = lane / LPH;
  Turn rot;
  load_turn(a, t, e0, lane, rot);
  float wq[8], wk[8];
  load_weights(a.wq, a.w32, e0, wq);
  load_weights(a.wk, a.w32, e0, wk);
  int64_t krow = (int64_t)t * a.ko.sl, vrow = (int64_t)t * a.vo.sl;
  bool kput = true;
  if (a.rows != nullptr) {
    const int row = a.rows[t];
    kput = row >= 0 && row < a.cap;
    krow = (int64_t)t * a.kosb + (int64_t)row * a.ko.sl;
    vrow = (int64_t)t * a.vosb + (int64_t)row * a.vo.sl;
  }
  const int nh = a.Hq + a.Hk, nall = nh + (a.v.p != nullptr ? a.Hk : 0);
  const int nch = (nall + HPW - 1) / HPW;
  for (int it = part; it < nch; it += U * a.parts) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = (it + u * a.parts) * HPW + hsub;
      const uint16_t* src = nullptr;
      if (hh < a.Hq) src = a.q.p + t * a.q.sl + hh * a.q.sh;
      else if (hh < nh) src = a.k.p + t * a.k.sl + (hh - a.Hq) * a.k.sh;
      else if (hh < nall) src = a.v.p + t * a.v.sl + (hh - nh) * a.v.sh;
      x[u] = u32x4{0u, 0u, 0u, 0u};
      if (src != nullptr) x[u] = load16(src + e0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if ((it + u * a.parts) >= nch) break;
      const int hh = (it + u * a.parts) * HPW + hsub;
      const bool is_q = hh < a.Hq;
      float f[8], y[8], o[8];
      unpack8(x[u], f);
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
      ss = head_sum<LPH>(ss);
      const float r = rsqrtf(ss * a.inv_d + a.eps) * (is_q ? a.q_scale : a.k_scale);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = f[j] * r * (is_q ? wq[j] : wk[j]);
      turn<false>(rot, a.inter, y, o);
      const u32x4 w = pack8(o);
      if (is_q)
        *reinterpret_cast<u32x4*>(a.qo.p + t * a.qo.sl + hh * a.qo.sh + e0) = w;
      else if (hh < nh && kput)
        *reinterpret_cast<u32x4*>(a.ko.p + krow + (hh - a.Hq) * a.ko.sh + e0) = w;
      else if (hh >= nh && hh < nall && kput)
        *reinterpret_cast<u32x4*>(a.vo.p + vrow + (hh - nh) * a.vo.sh + e0) = x[u];
    }
  }
}

// A workgroup's waves take tokens in turn (wave w of workgroup i: tokens 4 i + w, then every
// 4 nwg-th) and keep the weights' gradient of their lanes' values in registers; each workgroup
// writes one partial row, which the second kernel adds in a fixed order: no atomics.
template <int LPH>
__global__ void __launch_bounds__(HN_WAVES * 64) head_norm_bwd_kernel(const HeadNormArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH;
  constexpr int U = 2;
  __shared__ float red[HN_WAVES][2][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e0 = 8 * (lane % LPH), hsub = lane / LPH;
  float wq[8], wk[8], gq[8], gk[8];
  load_weights(a.wq, a.w32, e0, wq);
  load_weights(a.wk, a.w32, e0, wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) gq[j] = gk[j] = 0.0f;
  const int nh = a.Hq + a.Hk, nch = (nh + HPW - 1) / HPW;
  for (int64_t t = (int64_t)blockIdx.x * HN_WAVES + wave; t < a.T; t += (int64_t)a.nwg * HN_WAVES) {
    Turn rot;
    load_turn(a, (int)t, e0, lane, rot);
    for (int it = 0; it < nch; it += U) {
      u32x4 x[U], dy[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int hh = (it + u) * HPW + hsub;
        x[u] = dy[u] = u32x4{0u, 0u, 0u, 0u};
        if (hh < a.Hq) {
          x[u] = load16(a.q.p + t * a.q.sl + hh * a.q.sh + e0);
          dy[u] = load16(a.dqo.p + t * a.dqo.sl + hh * a.dqo.sh + e0);
        } else if (hh < nh) {
          x[u] = load16(a.k.p + t * a.k.sl + (hh - a.Hq) * a.k.sh + e0);
          dy[u] = load16(a.dko.p + t * a.dko.sl + (hh - a.Hq) * a.dko.sh + e0);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int hh = (it + u) * HPW + hsub;
        const bool is_q = hh < a.Hq;
        float f[8], d[8], g[8], o[8];
        unpack8(x[u], f);
        unpack8(dy[u], d);
        turn<true>(rot, a.inter, d, g);
        const float sc = is_q ? a.q_scale : a.k_scale;
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] *= sc;
          ss += f[j] * f[j];
          dot += g[j] * (is_q ? wq[j] : wk[j]) * f[j];
        }
        ss = head_sum<LPH>(ss);
        dot = head_sum<LPH>(dot);
        const float r = rsqrtf(ss * a.inv_d + a.eps);
        const float m = r * r * dot * a.inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float gx = g[j] * f[j] * r;
          if (is_q) gq[j] += gx;
          else if (hh < nh) gk[j] += gx;
          o[j] = r * (g[j] * (is_q ? wq[j] : wk[j]) - f[j] * m);
        }
        const u32x4 w = pack8(o);
        if (is_q)
          *reinterpret_cast<u32x4*>(a.qo.p + t * a.qo.sl + hh * a.qo.sh + e0) = w;
        else if (hh < nh)
          *reinterpret_cast<u32x4*>(a.ko.p + t * a.ko.sl + (hh - a.Hq) * a.ko.sh + e0) = w;
      }
    }
  }
  // lanes that hold the same values, then the waves
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 32; o >= LPH; o >>= 1) {
      gq[j] += __shfl_xor(gq[j], o);
      gk[j] += __shfl_xor(gk[j], o);
    }
  }
  if (lane < LPH) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      red[wave][0][e0 + j] = gq[j];
      red[wave][1][e0 + j] = gk[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += HN_WAVES * 64) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < HN_WAVES; ++w) s += red[w][i / D][i % D];
    a.part[(int64_t)blockIdx.x * 2 * D + i] = s;
  }
}

// The weights' gradient: the workgroups' partial rows added up, 32 columns per workgroup.
__global__ void __launch_bounds__(256) head_norm_dw_kernel(const HeadNormArgs a, int D) {
  __shared__ float red[8][32];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), strip = threadIdx.x >> 5;
  float s = 0.0f;
  for (int w = strip; w < a.nwg; w += 8) s += a.part[(int64_t)w * 2 * D + col];
  red[strip][threadIdx.x & 31] = s;
  __syncthreads();
  if (strip != 0) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
  void* dst = col < D ? a.dwq : a.dwk;
  if (dst == nullptr) return;
  if (a.w32) static_cast<float*>(dst)[col % D] = s;
  else static_cast<__bf16*>(dst)[col % D] = (__bf16)s;
}

template <int LPH>
hipError_t run_fwd(const HeadNormArgs& a, hipStream_t stream) {
  const int64_t waves = (int64_t)a.T * a.parts;
  hipLaunchKernelGGL((head_norm_kernel<LPH>), dim3((uint32_t)((waves + HN_WAVES - 1) / HN_WAVES)),
                     dim3(HN_WAVES * 64), 0, stream, a);
  return hipGetLastError();
}
template <int LPH>
hipError_t run_bwd(const HeadNormArgs& a, hipStream_t stream) {
  if (a.nwg > 0)
    hipLaunchKernelGGL((head_norm_bwd_kernel<LPH>), dim3(a.nwg), dim3(HN_WAVES * 64), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (a.dwq == nullptr && a.dwk == nullptr)) return e;
  hipLaunchKernelGGL(head_norm_dw_kernel, dim3(2 * 8 * LPH / 32), dim3(256), 0, stream, a, 8 * LPH);
  return hipGetLastError();
}

}  // namespace

// Workgroups of the gradient kernel: four per CU, or as many as the tokens fill.
int head_norm_bwd_workgroups(int T, int cus) {
  const int need = (T + HN_WAVES - 1) / HN_WAVES;
  return need < 4 * cus ? need : 4 * cus;
}

hipError_t launch_head_norm(const HeadNormArgs& args, int D, hipStream_t stream) {
  HeadNormArgs a = args;
  // a token's heads are shared by several waves while the tokens alone do not fill the chip
  const int nch = (a.Hq + 2 * a.Hk + 512 / D - 1) / (512 / D);
  a.parts = 1;
  while (a.parts < nch && (int64_t)a.T * a.parts < 4096) a.parts *= 2;
  switch (D) {
    case 32: return run_fwd<4>(a, stream);
    case 64: return run_fwd<8>(a, stream);
    case 128: return run_fwd<16>(a, stream);
    default: return run_fwd<32>(a, stream);
  }
}
hipError_t launch_head_norm_bwd(const HeadNormArgs& a, int D, hipStream_t stream) {
  switch (D) {
    case 32: return run_bwd<4>(a, stream);
    case 64: return run_bwd<8>(a, stream);
    case 128: return run_bwd<16>(a, stream);
    default: return run_bwd<32>(a, stream);
  }
}

}  // namespace lbw
