// Attention over packed sequences, forward (gfx950).
//
//   S = scale Q K^T over the keys j < k_len, j <= i + shift of query i's own sequence;
//   O = softmax(S) V, lse = ln sum_j exp(S); a query that sees no key gives O = 0, lse = -inf.
//
// One workgroup = 4 waves = 128 queries of one sequence and head; K and V stream through LDS in
// 64-key tiles, two stages each (64 KB), so two workgroups share a CU and one computes while the
// other waits. S^T = K Q^T and O^T = V^T P^T: a lane holds one query's column, so the softmax
// is lane-local but for one exchange with lane^32, and P^T goes from the accumulators straight into the
// second product. Online softmax in base 2 against a reference that moves when a row's sum in a
// step outgrows it.

#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int V_AT = 2 * PK_TILE_B;              // V stages behind the K stages
constexpr int FWD_LDS = 4 * PK_TILE_B;

__global__ void __launch_bounds__(PK_WAVES * 64, 2) packed_fwd_kernel(const PackedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  int h, kv;
  pick_head(blockIdx.x % (uint32_t)a.Hq, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, blockIdx.x / (uint32_t)a.Hq);
  if (!item_fits(it, a.Tq, a.Tk)) return;
  const int r0 = 32 * wave;                       // this wave's first row of the item
  const int rows = it.rows - r0;                  // and how many it has
  const bool active = rows > 0;

  u32x4 qf[8];
  if (active)
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

  const int lds0 = (int)lds_addr(lds);
  const int ka = row_address(lds0, l32, hl), va = tr_address(lds0 + V_AT, lane, hl);
  TileCopy copy;
  copy.init(wave, lane);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;

  floatx16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(o[db]);
  float m = M_INIT, l = 0.0f;
  const float c = a.scale_log2;
  const int T = (it.bound + BN - 1) / BN;
  if (T > 0) {
    copy.issue(kb, ks, 0, it.other_len, dst);
    copy.issue(vb, vs, 0, it.other_len, dst + V_AT);
  }
#pragma unroll 1
  for (int u = 0; u < T; ++u) {
    const int st = (u & 1) * PK_TILE_B;
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): its copies of tile u, its reads of u - 1
    barrier_nofence();                   // everybody's; and all are past tile u - 1
    if (u + 1 < T) {
      copy.issue(kb, ks, (u + 1) * BN, it.other_len, dst + (PK_TILE_B - st));
      copy.issue(vb, vs, (u + 1) * BN, it.other_len, dst + V_AT + (PK_TILE_B - st));
    }
    if (!active || u * BN >= lim_hi) continue;
#pragma unroll
    for (int kb32 = 0; kb32 < 2; ++kb32) {
      const int at = st + kb32 * 32 * PK_ROWB;
      floatx16 s;
      zero(s);
#pragma unroll
      for (int d = 0; d < 8; ++d) s = mfma32x32x16(read_row(ka, d, at), qf[d], s);
      const int key0 = u * BN + 32 * kb32;
      if (key0 + 32 > lim_lo) {
        const int left = lim - (key0 + 4 * hl);  // keys of this lane from register 0 on
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = acc_row(r) < left ? s[r] : -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
      mx = wave_max_xor32(mx);
      const float mn = fmaxf(m, mx);
      if (__any(mn > m)) {
        const float alpha = fast_exp2((m - mn) * c);
        scale_acc(o, alpha);
        l *= alpha;
        m = mn;
      }
      const float mc = -m * c;
      floatx16 p;
      float ls = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = fast_exp2(__builtin_fmaf(s[r], c, mc));
        ls += p[r];
      }
      l += ls;
      const u32x4 pf[2] = {pack_half(p, 0), pack_half(p, 1)};
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int mm = 0; mm < 2; ++mm) o[db] = mfma32x32x16(read_tr(va, db, mm, at), pf[mm], o[db]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();  // all waves are past their tile reads: the LDS is free for the output
  if (!active) return;
  l = wave_sum_xor32(l);
  if (a.lse != nullptr && hl == 0 && l32 < rows)
    a.lse[(int64_t)h * a.Tq + it.row0 + r0 + l32] = l > 0.0f ? m * a.scale + logf(l) : -INFINITY;
  store_rows(lds + 8192 * wave, o, l > 0.0f ? 1.0f / l : 0.0f, lane, rows, [&](int r) {
    return a.out.p + (int64_t)(it.row0 + r0 + r) * a.out.sl + h * a.out.sh;
  });
}

}  // namespace

hipError_t launch_packed_fwd(const PackedArgs& a, hipStream_t stream) {
  static hipError_t attr = hipFuncSetAttribute((const void*)packed_fwd_kernel,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, FWD_LDS);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL(packed_fwd_kernel, dim3((uint32_t)a.n_q_items * a.Hq), dim3(PK_WAVES * 64),
                     FWD_LDS, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
