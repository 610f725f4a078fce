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
// registers (cos and signed sin of the lane's eight values) and serve all its heads. 32759 tokens x 12 + 12
// heads of 128: forward 66.7 us (6.0 TB/s), gradient 134.7 us (4.5 TB/s; a large copy reaches 4.9);
// one token 4.8 us, most of it the launch.

#include "common.h"
#include "packed.h"

namespace lbw {
namespace {

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

template <bool INTER>
__device__ __forceinline__ void load_turn(const HeadNormArgs& a, int t, int e0, int lane, Turn& r) {
  const int h = a.npairs;
  // the token's positions (selected by comparisons: an array would be put into LDS)
  const int32_t* pos = a.pos + (int64_t)t * a.pos_sl;
  const int p0 = pos[0], p1 = a.naxes > 1 ? pos[1] : 0, p2 = a.naxes > 2 ? pos[2] : 0,
            p3 = a.naxes > 3 ? pos[3] : 0;
  auto angle = [&](int i) {
    const int lo = i >= a.ax_end[0] ? p1 : p0, hi = i >= a.ax_end[2] ? p3 : p2;
    const int p = i >= a.ax_end[1] ? hi : lo;
    float2 cs = {1.0f, 0.0f};
    if (i < h) {  // a position outside the table turns by NaN
      cs = {__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u)};
      if (p >= 0 && p < a.P) cs = a.table[(int64_t)p * h + i];
    }
    return cs;
  };
  r.lane = lane;
  if constexpr (INTER) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 cs = angle((e0 >> 1) + j);
      r.c[2 * j] = r.c[2 * j + 1] = cs.x;
      r.s[2 * j] = -cs.y;
      r.s[2 * j + 1] = cs.y;
    }
  } else {
    const bool second = e0 >= h;
    if (e0 < 2 * h) r.lane = second ? lane - h / 8 : lane + h / 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 cs = angle(second ? e0 + j - h : e0 + j);
      r.c[j] = cs.x;
      r.s[j] = second ? cs.y : -cs.y;
    }
  }
}

// y turned; back: by the negative angle.
template <bool INTER, bool BACK>
__device__ __forceinline__ void turn(const Turn& r, const float (&y)[8], float (&o)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float p = INTER ? y[j ^ 1] : __shfl(y[j], r.lane);
    o[j] = y[j] * r.c[j] + p * (BACK ? -r.s[j] : r.s[j]);
  }
}

// One tensor of a token: chunk i holds heads i HPW .. (lane / LPH counts them). Element offsets of a lane
// within a chunk fit 32 bits (the host checks); the chunk's base is scalar.
struct Lane {
  int e0, hsub;
};

// Chunks first, first + step, .. of `heads` heads: normed and turned (w, scale), or copied.
template <int LPH, bool INTER, bool COPY>
__device__ __forceinline__ void norm_rows(const uint16_t* src, int64_t ssh, uint16_t* dst, int64_t dsh,
                                          int heads, int first, int step, Lane ln, const void* w,
                                          int w32, float scale, const Turn& rot, float inv_d, float eps) {
  constexpr int HPW = 64 / LPH, U = 4;
  const int nch = (heads + HPW - 1) / HPW;
  if (first >= nch) return;
  const uint32_t so = (uint32_t)(ln.hsub * (int)ssh + ln.e0), dof = (uint32_t)(ln.hsub * (int)dsh + ln.e0);
  float wt[8];
  if constexpr (!COPY) load_weights(w, w32, ln.e0, wt);
  for (int it = first; it < nch; it += U * step) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      x[u] = u32x4{0u, 0u, 0u, 0u};
      if (ch * HPW + ln.hsub < heads) x[u] = load16(src + (int64_t)ch * HPW * ssh + so);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ch = it + u * step;
      if (ch >= nch) break;
      u32x4 out = x[u];
      if constexpr (!COPY) {
        float f[8], o[8];
        unpack8(x[u], f);
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
        const float r = rsqrtf(head_sum<LPH>(ss) * inv_d + eps) * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= r * wt[j];
        turn<INTER, false>(rot, f, o);
        out = pack8(o);
      }
      if (dst != nullptr && ch * HPW + ln.hsub < heads)
        *reinterpret_cast<u32x4*>(dst + (int64_t)ch * HPW * dsh + dof) = out;
    }
  }
}

template <int LPH, bool INTER>
__global__ void __launch_bounds__(HN_WAVES * 64) head_norm_kernel(const HeadNormArgs a) {
  constexpr int HPW = 64 / LPH;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * HN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tt = id / a.parts;
  if (tt >= a.T) return;
  const int t = (int)tt, part = (int)(id % a.parts);
  const Lane ln = {8 * (lane % LPH), lane / LPH};
  Turn rot;
  load_turn<INTER>(a, t, ln.e0, lane, rot);
  uint16_t *ko = a.ko.p + (int64_t)t * a.ko.sl, *vo = a.vo.p + (int64_t)t * a.vo.sl;
  if (a.rows != nullptr) {
    const int row = __builtin_amdgcn_readfirstlane(a.rows[t]);
    const bool put = row >= 0 && row < a.cap;
    ko = put ? a.ko.p + (int64_t)t * a.kosb + (int64_t)row * a.ko.sl : nullptr;
    vo = put ? a.vo.p + (int64_t)t * a.vosb + (int64_t)row * a.vo.sl : nullptr;
  }
  // the token's chunks, q's, k's, v's, in turn to the waves that share it
  const int cq = (a.Hq + HPW - 1) / HPW, ck = (a.Hk + HPW - 1) / HPW;
  auto first = [&](int before) {
    const int x = (part - before) % a.parts;
    return x < 0 ? x + a.parts : x;
  };
  norm_rows<LPH, INTER, false>(a.q.p + t * a.q.sl, a.q.sh, a.qo.p + t * a.qo.sl, a.qo.sh, a.Hq, part, a.parts,
                               ln, a.wq, a.w32, a.q_scale, rot, a.inv_d, a.eps);
  norm_rows<LPH, INTER, false>(a.k.p + t * a.k.sl, a.k.sh, ko, a.ko.sh, a.Hk, first(cq), a.parts, ln, a.wk,
                               a.w32, a.k_scale, rot, a.inv_d, a.eps);
  if (a.v.p != nullptr)
    norm_rows<LPH, INTER, true>(a.v.p + t * a.v.sl, a.v.sh, vo, a.vo.sh, a.Hk, first(cq + ck), a.parts, ln,
                                nullptr, 0, 1.0f, rot, a.inv_d, a.eps);
}

// Workgroups 0 .. nwg_q - 1 take q, the others k, in proportion to their heads. A workgroup's waves take
// tokens in turn and keep the weights' gradient of their lanes' values in registers; each workgroup writes
// one partial row, which the second kernel adds in a fixed order: no atomics.
template <int LPH, bool INTER>
__global__ void __launch_bounds__(HN_WAVES * 64) head_norm_bwd_kernel(const HeadNormArgs a) {
  constexpr int HPW = 64 / LPH, D = 8 * LPH, U = 2;
  __shared__ float red[HN_WAVES][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = 8 * (lane % LPH), hsub = lane / LPH;
  const bool is_q = (int)blockIdx.x < a.nwg_q;
  const int wg = is_q ? blockIdx.x : blockIdx.x - a.nwg_q, nwg = is_q ? a.nwg_q : a.nwg - a.nwg_q;
  const Rows src = is_q ? a.q : a.k, grad = is_q ? a.dqo : a.dko;
  const RowsOut dst = is_q ? a.qo : a.ko;
  const int heads = is_q ? a.Hq : a.Hk, nch = (heads + HPW - 1) / HPW;
  const float scale = is_q ? a.q_scale : a.k_scale;
  const uint32_t so = (uint32_t)(hsub * (int)src.sh + e0), go = (uint32_t)(hsub * (int)grad.sh + e0),
                 dof = (uint32_t)(hsub * (int)dst.sh + e0);
  float wt[8], gw[8];
  load_weights(is_q ? a.wq : a.wk, a.w32, e0, wt);
#pragma unroll
  for (int j = 0; j < 8; ++j) gw[j] = 0.0f;
  for (int64_t t = (int64_t)wg * HN_WAVES + wave; t < a.T; t += (int64_t)nwg * HN_WAVES) {
    const uint16_t *xs = src.p + t * src.sl, *gs = grad.p + t * grad.sl;
    uint16_t* ds = dst.p + t * dst.sl;
    u32x4 x[U], dy[U];
    auto load = [&](int it) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = dy[u] = u32x4{0u, 0u, 0u, 0u};
        if ((it + u) * HPW + hsub < heads) {
          x[u] = load16(xs + (int64_t)(it + u) * HPW * src.sh + so);
          dy[u] = load16(gs + (int64_t)(it + u) * HPW * grad.sh + go);
        }
      }
    };
    load(0);  // ahead of the table, whose rows depend on the positions
    Turn rot;
    load_turn<INTER>(a, (int)t, e0, lane, rot);
    for (int it = 0; it < nch; it += U) {
      if (it != 0) load(it);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[8], g[8], o[8];
        unpack8(dy[u], f);
        turn<INTER, true>(rot, f, g);
        unpack8(x[u], f);
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] *= scale;
          ss += f[j] * f[j];
          dot += g[j] * wt[j] * f[j];
        }
        ss = head_sum<LPH>(ss);
        dot = head_sum<LPH>(dot);
        const bool there = (it + u) * HPW + hsub < heads;
        // (a lane past the last head holds zeros, and with eps = 0 their rsqrt is infinite)
        const float r = there ? rsqrtf(ss * a.inv_d + a.eps) : 0.0f;
        const float m = r * r * dot * a.inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          gw[j] += g[j] * f[j] * r;
          o[j] = r * (g[j] * wt[j] - f[j] * m);
        }
        if (there)
          *reinterpret_cast<u32x4*>(ds + (int64_t)(it + u) * HPW * dst.sh + dof) = pack8(o);
      }
    }
  }
  // lanes that hold the same values, then the waves
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 32; o >= LPH; o >>= 1) gw[j] += __shfl_xor(gw[j], o);
  }
  if (lane < LPH) {
#pragma unroll
    for (int j = 0; j < 8; ++j) red[wave][e0 + j] = gw[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += HN_WAVES * 64) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < HN_WAVES; ++w) s += red[w][i];
    a.part[(int64_t)blockIdx.x * D + i] = s;
  }
}

// The weights' gradient: the workgroups' partial rows added up in a fixed order, 16 columns per
// workgroup, 64 strips of rows.
__global__ void __launch_bounds__(1024) head_norm_dw_kernel(const HeadNormArgs a, int D) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, strip = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  const int w0 = col < D ? 0 : a.nwg_q, w1 = col < D ? a.nwg_q : a.nwg;
  float s = 0.0f;
#pragma unroll 8
  for (int w = w0 + strip; w < w1; w += 64) s += a.part[(int64_t)w * D + col % D];
  red[strip][c] = s;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    __syncthreads();
    if (strip < o) red[strip][c] += red[strip + o][c];
  }
  if (strip != 0) return;
  s = red[0][c];
  void* dst = col < D ? a.dwq : a.dwk;
  if (dst == nullptr) return;
  if (a.w32) static_cast<float*>(dst)[col % D] = s;
  else static_cast<__bf16*>(dst)[col % D] = (__bf16)s;
}

template <int LPH>
hipError_t run_fwd(const HeadNormArgs& a, hipStream_t stream) {
  const int64_t waves = (int64_t)a.T * a.parts;
  const dim3 grid((uint32_t)((waves + HN_WAVES - 1) / HN_WAVES)), block(HN_WAVES * 64);
  if (a.inter) hipLaunchKernelGGL((head_norm_kernel<LPH, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((head_norm_kernel<LPH, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}
template <int LPH>
hipError_t run_bwd(const HeadNormArgs& a, hipStream_t stream) {
  const dim3 grid(a.nwg), block(HN_WAVES * 64);
  if (a.nwg > 0) {
    if (a.inter) hipLaunchKernelGGL((head_norm_bwd_kernel<LPH, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((head_norm_bwd_kernel<LPH, false>), grid, block, 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (a.dwq == nullptr && a.dwk == nullptr)) return e;
  hipLaunchKernelGGL(head_norm_dw_kernel, dim3(2 * 8 * LPH / 16), dim3(1024), 0, stream, a, 8 * LPH);
  return hipGetLastError();
}

}  // namespace

// Workgroups of the gradient kernel: four per CU, or as many as the tokens fill (for q and for k).
int head_norm_bwd_workgroups(int T, int cus) {
  const int64_t need = 2 * (((int64_t)T + HN_WAVES - 1) / HN_WAVES);
  return need < 4 * cus ? (int)need : 4 * cus;
}

hipError_t launch_head_norm(const HeadNormArgs& args, int D, hipStream_t stream) {
  HeadNormArgs a = args;
  // a token's heads are shared by several waves while the tokens alone do not fill the chip
  const int nch = (a.Hq + 2 * a.Hk + 512 / D - 1) / (512 / D);
  a.parts = 1;
  while (a.parts < nch && (int64_t)a.T * a.parts < 16384) a.parts *= 2;
  switch (D) {
    case 32: return run_fwd<4>(a, stream);
    case 64: return run_fwd<8>(a, stream);
    case 128: return run_fwd<16>(a, stream);
    default: return run_fwd<32>(a, stream);
  }
}
hipError_t launch_head_norm_bwd(const HeadNormArgs& args, int D, hipStream_t stream) {
  HeadNormArgs a = args;
  a.nwg_q = (int)((int64_t)a.nwg * a.Hq / (a.Hq + a.Hk));  // (k has at most q's heads: never all)
  switch (D) {
    case 32: return run_bwd<4>(a, stream);
    case 64: return run_bwd<8>(a, stream);
    case 128: return run_bwd<16>(a, stream);
    default: return run_bwd<32>(a, stream);
  }
}

}  // namespace lbw
