// Attention over packed sequences, forward (gfx950).
//
//   S = scale Q K^T over the keys j < k_len, j <= i + shift of query i's own sequence;
//   O = softmax(S) V, lse = ln sum_j exp(S); a query that sees no key gives O = 0, lse = -inf.
//
// A group of 4 waves takes 128 queries of one sequence and head; K and V stream through LDS in
// 64-key tiles, two stages each (64 KB a group). S^T = K Q^T and O^T = V^T P^T: a lane holds one
// query's column, so the softmax is lane-local but for one exchange with lane^32, and P^T goes from the
// accumulators straight into the second product.
//
// Software pipeline (per wave, 32-key blocks): the softmax of block j (VALU) runs beside the MFMAs of
// O += V_{j-1}^T P_{j-1}^T and S_{j+1} = K_{j+1} Q^T. Online softmax in base 2 against a reference
// that moves only when a row's sum in a step outgrows it; O and l share it, so the result is exact.

#include <stdlib.h>
#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int V_AT = 2 * PK_TILE_B;              // V stages behind the K stages
constexpr int GROUP_B = 4 * PK_TILE_B;           // LDS of a group of 4 waves
constexpr int HALF_B = PK_TILE_B / 2;
constexpr int AHEAD = 2;                         // MFMA pairs that LDS fragments are read ahead

template <int N>
using ic = std::integral_constant<int, N>;

// GROUPS = 1: a workgroup is one group, two workgroups share a CU. GROUPS = 2: two groups share a work
// item, each with half of its keys, and join their results in LDS.
template <int GROUPS>
__global__ void __launch_bounds__(GROUPS * PK_WAVES * 64, GROUPS == 1 ? 2 : 1)
packed_fwd_kernel(const PackedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_id % PK_WAVES, grp = wave_id / PK_WAVES;
  const int hl = lane >> 5, l32 = lane & 31;
  int h, kv;
  pick_head(blockIdx.x % (uint32_t)a.Hq, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, blockIdx.x / (uint32_t)a.Hq);
  if (!item_fits(it, a.Tq, a.Tk)) return;
  const int r0 = 32 * wave;                       // this wave's first row of the item
  const int rows = it.rows - r0;                  // and how many it has

  u32x4 qf[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) qf[s] = u32x4{0u, 0u, 0u, 0u};
  if (rows > 0)
    load_rows(a.q.p + (int64_t)(it.row0 + r0) * a.q.sl + h * a.q.sh, a.q.sl, rows, l32, hl, qf);
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(
      a.k.p + (int64_t)it.other0 * a.k.sl + kv * a.k.sh);
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(
      a.v.p + (int64_t)it.other0 * a.v.sl + kv * a.v.sh);
  const int64_t ks = a.k.sl * 2, vs = a.v.sl * 2;

  // keys that this lane's query sees, and the wave's smallest and largest such count
  const int i0 = it.pos0 + r0;
  auto limit = [&](int i) {
    const int64_t x = (int64_t)i + it.shift + 1;
    return (int)(x < 0 ? 0 : (x < it.other_len ? x : it.other_len));
  };
  const int lim = limit(i0 + l32);
  const int lim_lo = limit(i0), lim_hi = limit(i0 + (rows < 32 ? rows : 32) - 1);
  // this group's tiles [t0, t0 + T) of the item, of which this wave needs the first Tw; the loop
  // runs Tmax times in every wave of the workgroup
  const int n_tiles = (it.bound + BN - 1) / BN;
  const int t0 = n_tiles * grp / GROUPS, T = n_tiles * (grp + 1) / GROUPS - t0;
  const int Tmax = (n_tiles + GROUPS - 1) / GROUPS;
  int Tw = rows > 0 ? (lim_hi + BN - 1) / BN - t0 : 0;
  Tw = Tw < 0 ? 0 : (Tw < T ? Tw : T);

  const int lds0 = (int)lds_addr(lds) + GROUP_B * grp;
  const int ka = row_address(lds0, l32, hl), va = tr_address(lds0 + V_AT, lane, hl);
  TileCopy copy;
  copy.init(wave, lane);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;
  auto issue_k = [&](int u) { copy.issue(kb, ks, (t0 + u) * BN, it.other_len, dst + (u & 1) * PK_TILE_B); };
  auto issue_v = [&](int u) {
    copy.issue(vb, vs, (t0 + u) * BN, it.other_len, dst + V_AT + (u & 1) * PK_TILE_B);
  };

  floatx16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(o[db]);
  float m = M_INIT, l = 0.0f;
  const float c = sreg(a.scale_log2);

  if (Tmax > 0) {
    if (T > 0) {
      issue_k(0);
      issue_v(0);
      if (T > 1) issue_k(1);
    }
    // the first step's "previous block" is the second half of V stage 1, with P = 0: zeros there
    *reinterpret_cast<u32x4*>(lds + GROUP_B * grp + V_AT + PK_TILE_B + HALF_B + 1024 * 2 * wave + 16 * lane) =
        u32x4{0u, 0u, 0u, 0u};
    *reinterpret_cast<u32x4*>(lds + GROUP_B * grp + V_AT + PK_TILE_B + HALF_B + 1024 * (2 * wave + 1) + 16 * lane) =
        u32x4{0u, 0u, 0u, 0u};
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    barrier_nofence();
  }

  floatx16 sA, sB;
  zero(sA);
  zero(sB);
  u32x4 pA[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  u32x4 pB[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  constexpr int R = AHEAD + 2;  // fragments of pair i in slot i % R (8 % R == 0)
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + AHEAD < 8) {
        load_k(ko, i + AHEAD);
        load_v(vo, i + AHEAD);
      }
      s_out = mfma32x32x16(kf[i % R], qf[i], s_out);
      o[i >> 1] = mfma32x32x16(vf[i % R], p_in[i & 1], o[i >> 1]);
    }
    auto exps = [&]() {
      float ls = 0.0f;
#pragma unroll
      for (int mm = 0; mm < 2; ++mm)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = fast_exp2(__builtin_fmaf(s_in[8 * mm + 2 * e], c, mc));
          const float x1 = fast_exp2(__builtin_fmaf(s_in[8 * mm + 2 * e + 1], c, mc));
          p_out[mm][e] = pack_bf16x2(x0, x1);
          ls += x0 + x1;
        }
      return ls;
    };
    float ls = exps();
    // the step's order: the first fragments, then MFMA, 2 VALU, fragments AHEAD pairs on, MFMA, 2 VALU
    __builtin_amdgcn_sched_group_barrier(0x100, 3 * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      if (i + AHEAD < 8) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
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
      ls = exps();
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
  for (int u = 0; u < Tmax; u += 2) {
    tile(ic<0>{}, u);
    if (u + 1 < Tmax) tile(ic<1>{}, u + 1);
  }
  if (Tw == Tmax && Tw > 0) drain(Tw - 1);
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();  // all waves are past their tile reads: the LDS is free for the output
  float ls = wave_sum_xor32(l);
  if constexpr (GROUPS == 2) {
    // group 1 hands its O, m and l over in register order, 16 bytes per lane
    unsigned char* og = lds + GROUP_B + 16384 * wave + 16 * lane;
    float* ml = reinterpret_cast<float*>(lds + 32768 + 512 * wave);
    if (grp == 1) {
#pragma unroll
      for (int x = 0; x < 16; ++x)
        *reinterpret_cast<floatx4*>(og + 1024 * x) =
            floatx4{o[x >> 2][4 * (x & 3)], o[x >> 2][4 * (x & 3) + 1], o[x >> 2][4 * (x & 3) + 2],
                    o[x >> 2][4 * (x & 3) + 3]};
      ml[lane] = m;
      ml[64 + lane] = ls;
    }
    __syncthreads();
    if (grp == 1) return;
    const float m1 = ml[lane], l1 = ml[64 + lane];
    const float mn = fmaxf(m, m1);  // (a half without keys: M_INIT, l = 0, O = 0)
    const float f0 = fast_exp2((m - mn) * c), f1 = fast_exp2((m1 - mn) * c);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const floatx4 y = *reinterpret_cast<const floatx4*>(og + 1024 * x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float& z = reinterpret_cast<float*>(&o[x >> 2])[4 * (x & 3) + e];
        z = z * f0 + y[e] * f1;
      }
    }
    ls = ls * f0 + l1 * f1;
    m = mn;
  }
  if (rows <= 0) return;
  if (a.lse != nullptr && hl == 0 && l32 < rows)
    a.lse[(int64_t)h * a.Tq + it.row0 + r0 + l32] = ls > 0.0f ? m * a.scale + logf(ls) : -INFINITY;
  store_rows(lds + 8192 * wave, o, ls > 0.0f ? 1.0f / ls : 0.0f, lane, rows, [&](int r) {
    return a.out.p + (int64_t)(it.row0 + r0 + r) * a.out.sl + h * a.out.sh;
  });
}

template <int GROUPS>
hipError_t run(const PackedArgs& a, hipStream_t stream) {
  static hipError_t attr = hipFuncSetAttribute((const void*)packed_fwd_kernel<GROUPS>,
                                               hipFuncAttributeMaxDynamicSharedMemorySize,
                                               GROUPS * GROUP_B);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL(packed_fwd_kernel<GROUPS>, dim3((uint32_t)a.n_q_items * a.Hq),
                     dim3(GROUPS * PK_WAVES * 64), GROUPS * GROUP_B, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_fwd(const PackedArgs& a, hipStream_t stream) {
  const char* e = getenv("LBW_G");
  return e && e[0] == '3' ? run<2>(a, stream) : run<1>(a, stream);
}

}  // namespace lbw
