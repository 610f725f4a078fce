// Rows of heads, eight values a lane (per-head norm, append to a paged cache): D / 8 lanes hold a head, a wave
// 512 / D heads.
#pragma once

#include "common.h"
#include "packed.h"

namespace lbw {

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

// `a` holds the table and the pairs of each axis; p0 .. p3: the token's positions (selected by comparisons: an
// array would be put into LDS).
template <bool INTER, typename Args>
__device__ __forceinline__ void load_turn_at(const Args& a, int p0, int p1, int p2, int p3, int e0, int lane,
                                             Turn& r) {
  const int h = a.npairs;
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

template <bool INTER, typename Args>
__device__ __forceinline__ void load_turn(const Args& a, int t, int e0, int lane, Turn& r) {
  const int32_t* pos = a.pos + (int64_t)t * a.pos_sl;
  load_turn_at<INTER>(a, pos[0], a.naxes > 1 ? pos[1] : 0, a.naxes > 2 ? pos[2] : 0, a.naxes > 3 ? pos[3] : 0,
                      e0, lane, r);
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

}  // namespace lbw
