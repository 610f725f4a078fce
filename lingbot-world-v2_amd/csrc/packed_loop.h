// The walk of a workgroup of 4 waves, 32 query rows each, over 64-key tiles of K and V (packed attention forward, the
// common prefix of a paged batch): scores, online softmax and output, the tiles' copies being the caller's.
#pragma once

#include <type_traits>

#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int V_AT = 2 * PK_TILE_B;              // V stages behind the K stages
constexpr int FWD_LDS = 4 * PK_TILE_B;
constexpr int HALF_B = PK_TILE_B / 2;
constexpr int AHEAD = 2;                         // MFMA pairs that LDS fragments are read ahead

template <int N>
using ic = std::integral_constant<int, N>;

// The first tiles on their way, and there.
template <typename IssueK, typename IssueV>
__device__ __forceinline__ void first_tiles(unsigned char* lds, int wave, int lane, int T, IssueK& issue_k,
                                            IssueV& issue_v) {
  issue_k(0);
  issue_v(0);
  if (T > 1) issue_k(1);
  // the first step's "previous block" is the second half of V stage 1, with P = 0: zeros there
  unsigned char* const zv = lds + V_AT + PK_TILE_B + HALF_B + 2048 * wave + 16 * lane;
  *reinterpret_cast<u32x4*>(zv) = u32x4{0u, 0u, 0u, 0u};
  *reinterpret_cast<u32x4*>(zv + 1024) = u32x4{0u, 0u, 0u, 0u};
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  barrier_nofence();
}

// A wave without rows: its share of the copies, in step with the others of its workgroup.
template <typename IssueK, typename IssueV>
__device__ __forceinline__ void copy_tiles(unsigned char* lds, int wave, int lane, int T, IssueK issue_k,
                                           IssueV issue_v) {
  if (T > 0) first_tiles(lds, wave, lane, T, issue_k, issue_v);
#pragma unroll 1
  for (int u = 0; u < T; ++u) {
    __builtin_amdgcn_s_waitcnt(0x0070);
    barrier_nofence();
    if (u + 2 < T) issue_k(u + 2);
    if (u + 1 < T) issue_v(u + 1);
  }
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();
}

// O^T, the reference m and the sum l (of the lane's half of the keys) of the wave's rows `qf` over tiles t0 .. t0 + T - 1,
// of which the wave needs the first Tw. A lane's row sees keys below `lim`, all of the wave's rows those below lim_lo.
// issue_k(u), issue_v(u): the wave's share of tile t0 + u on its way into stage u % 2. On return all waves are past
// their tile reads.
template <typename IssueK, typename IssueV>
__device__ __forceinline__ void attend_tiles(unsigned char* lds, int wave, int lane, const u32x4 (&qf)[8], float c, int t0,
                                             int T, int Tw, int lim, int lim_lo, IssueK issue_k, IssueV issue_v,
                                             floatx16 (&o)[4], float& m, float& l) {
  const int lds0 = (int)lds_addr(lds), hl = lane >> 5, l32 = lane & 31;
  const int ka = row_address(lds0, l32, hl), va = tr_address(lds0 + V_AT, lane, hl);
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(o[db]);
  m = M_INIT;
  l = 0.0f;

  if (T > 0) first_tiles(lds, wave, lane, T, issue_k, issue_v);

  floatx16 sA, sB;
  zero(sA);
  zero(sB);
  u32x4 pA[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  u32x4 pB[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  constexpr int R = AHEAD + 1;  // fragments of pair i in slot i % R
  u32x4 kf[R], vf[R];
  auto load_k = [&](auto ko, int i) { kf[i % R] = read_row(ka, i, decltype(ko)::value); };
  auto load_v = [&](auto vo, int i) { vf[i % R] = read_tr(va, i >> 1, i & 1, decltype(vo)::value); };

  if (Tw > 0) {
#pragma unroll
    for (int d = 0; d < 8; ++d) sA = mfma32x32x16(read_row(ka, d, 0), qf[d], sA);
  }

  // One step: softmax of s_in (keys key0 ..) into p_out, O += V^T p_in^T from V offset VO, s_out = K Q^T
  // from K offset KO.
  auto step = [&](auto ko, auto vo, floatx16& s_in, floatx16& s_out, u32x4 (&p_in)[2],
                  u32x4 (&p_out)[2], int key0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      load_k(ko, i);
      load_v(vo, i);
    }
    if (key0 + 32 > lim_lo) {
      const int left = lim - (key0 + 4 * hl);  // keys of this lane from register 0 on
#pragma unroll
      for (int r = 0; r < 16; ++r) s_in[r] = acc_row(r) < left ? s_in[r] : -INFINITY;
    }
    float mc = -m * c;
    zero(s_out);
    float ls = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + AHEAD < 8) {
        load_k(ko, i + AHEAD);
        load_v(vo, i + AHEAD);
      }
      s_out = mfma32x32x16(kf[i % R], qf[i], s_out);
      const float x0 = fast_exp2(__builtin_fmaf(s_in[2 * i], c, mc));
      const float x1 = fast_exp2(__builtin_fmaf(s_in[2 * i + 1], c, mc));
      o[i >> 1] = mfma32x32x16(vf[i % R], p_in[i & 1], o[i >> 1]);
      p_out[i >> 2][i & 3] = pack_bf16x2(x0, x1);  // registers 2 i, 2 i + 1: word i of the operand
      ls += x0 + x1;
      // (two products and two exponentials a pair, in this order)
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" ::"v"(p_out[0]), "v"(p_out[1]), "v"(ls));
    // a sum past the limit (or not finite): some p outgrew the reference. Move it to the row's max
    // and redo; O (with this step's product, at the old reference) and l follow.
    if (__any(!(ls <= P_LIMIT))) {
      float mx = s_in[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s_in[r]);
      mx = wave_max_xor32(mx);
      const float mn = fmaxf(mx, m);
      const float alpha = fast_exp2((m - mn) * c);
      m = mn;
      mc = -mn * c;
      scale_acc(o, alpha);
      l *= alpha;
      ls = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = fast_exp2(__builtin_fmaf(s_in[2 * i], c, mc));
        const float x1 = fast_exp2(__builtin_fmaf(s_in[2 * i + 1], c, mc));
        p_out[i >> 2][i & 3] = pack_bf16x2(x0, x1);
        ls += x0 + x1;
      }
    }
    l += ls;
    asm volatile("" ::"v"(p_out[0]), "v"(p_out[1]), "v"(l));
  };
  // O += V^T P^T of the wave's last block (its second half, P in pA)
  auto drain = [&](int u) {
    const int at = (u & 1) * PK_TILE_B + HALF_B;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i >> 1] = mfma32x32x16(read_tr(va, i >> 1, i & 1, at), pA[i & 1], o[i >> 1]);
  };

  // Tile u: stage u % 2 of K and of V. Step 2u: softmax of its first half, PV of tile u - 1's second
  // half, S of its second half. Then tile u's V and tile u + 1's K have to be there, and every wave is
  // past K tile u and V tile u - 1, whose stages take K tile u + 2 and V tile u + 1. Step 2u + 1:
  // softmax of its second half, PV of its first, S of tile u + 1's first half.
  auto tile = [&](auto st_c, int u) {
    constexpr int ST = decltype(st_c)::value, SN = 1 - ST;
    const int key0 = (t0 + u) * BN;
    if (u < Tw)
      step(ic<ST * PK_TILE_B + HALF_B>{}, ic<SN * PK_TILE_B + HALF_B>{}, sA, sB, pA, pB, key0);
    else if (u == Tw && Tw > 0)
      drain(u - 1);
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): its copies, its reads
    barrier_nofence();
    if (u + 2 < T) issue_k(u + 2);
    if (u + 1 < T) issue_v(u + 1);
    if (u < Tw) step(ic<SN * PK_TILE_B>{}, ic<ST * PK_TILE_B>{}, sB, sA, pB, pA, key0 + 32);
  };
#pragma unroll 1
  for (int u = 0; u < T; u += 2) {
    tile(ic<0>{}, u);
    if (u + 1 < T) tile(ic<1>{}, u + 1);
  }
  if (Tw == T && Tw > 0) drain(Tw - 1);
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();  // all waves are past their tile reads: the LDS is free for the output
}

}  // namespace
}  // namespace lbw
