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
//
// P goes to bf16 as the second product's operand: one rounding of each weight, which l does not see.
//
// 4680 + 3600 + 1561 causal tokens x 40/8 heads 394 us, 970 TFLOP/s (a library product of 16384^3 reaches 1364);
// the MFMA pipes are busy 55 % of the cycles at 1.65 GHz. That is not their limit: on the same products (3600 rows
// over 46800 keys x 40 heads, full, one run) the chunk attention kernel keeps them busy 65 % of the cycles at 1.70
// GHz, this one 58 % at 1.51 GHz (3278 / 4121 us). It has 17 % fewer vector instructions, three stages and counted
// waits where this one waits for all copies at every tile, and 256 queries to a tile of K and V where this one has
// 128; which of these costs what is not measured. Two workgroups a CU hide each other's barriers: one of eight
// waves, half the keys to each four, in step, took 522 us where two of four waves took 437.

#include "capi_util.h"
#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int V_AT = 2 * PK_TILE_B;              // V stages behind the K stages
constexpr int FWD_LDS = 4 * PK_TILE_B;
constexpr int HALF_B = PK_TILE_B / 2;
constexpr int AHEAD = 2;                         // MFMA pairs that LDS fragments are read ahead

template <int N>
using ic = std::integral_constant<int, N>;

// A wave's rows of lse from the reference and the sum (of both lane halves): -inf for a sum of 0, a row that sees
// no key; a sum that is NaN stays NaN.
__device__ __forceinline__ void store_lse(const PackedArgs& a, int h, int64_t row0, int lane, int rows, float m,
                                          float l) {
  if (a.lse != nullptr && lane < 32 && lane < rows)
    a.lse[(int64_t)h * a.Tq + row0 + lane] = l == 0.0f ? -INFINITY : m * a.scale + logf(l);
}

__global__ void __launch_bounds__(PK_WAVES * 64, 2) packed_fwd_kernel(const PackedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  int h, kv;
  const PackedShare sh = pick_share(a, blockIdx.x, a.Hq);
  pick_head(sh.head, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, sh.item);
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
  // this piece's tiles [t0, t0 + T), of which this wave needs the first Tw
  const int n_tiles = (it.bound + BN - 1) / BN, pieces = pieces_of(a, sh, n_tiles);
  if (sh.piece >= pieces) return;
  const int t0 = (int)((int64_t)n_tiles * sh.piece / pieces);
  const int T = (int)((int64_t)n_tiles * (sh.piece + 1) / pieces) - t0;
  int Tw = rows > 0 ? (lim_hi + BN - 1) / BN - t0 : 0;
  Tw = Tw < 0 ? 0 : (Tw < T ? Tw : T);

  const int lds0 = (int)lds_addr(lds);
  const int ka = row_address(lds0, l32, hl), va = tr_address(lds0 + V_AT, lane, hl);
  TileCopy copy;
  copy.init(wave, lane);
  const uint32_t koff = copy.row_offset(ks), voff = copy.row_offset(vs);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;
  auto issue_k = [&](int u) { copy.issue(kb, ks, koff, (t0 + u) * BN, it.other_len, dst + (u & 1) * PK_TILE_B); };
  auto issue_v = [&](int u) {
    copy.issue(vb, vs, voff, (t0 + u) * BN, it.other_len, dst + V_AT + (u & 1) * PK_TILE_B);
  };

  floatx16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(o[db]);
  float m = M_INIT, l = 0.0f;
  const float c = sreg(a.scale_log2);

  if (T > 0) {
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
  if (rows <= 0) return;
  const float ls = wave_sum_xor32(l);
  if (pieces > 1) {
    float* const part = part_of(a, sh, a.Hq, sh.piece, PK_PART_FWD);
    store_acc(part, wave, lane, o);
    if (hl == 0) {
      part[PK_BLOCK * 128 + r0 + l32] = ls == 0.0f ? -INFINITY : m;
      part[PK_BLOCK * 128 + PK_BLOCK + r0 + l32] = ls;
    }
    return;
  }
  const int64_t row0 = it.row0 + 32 * wave;
  store_lse(a, h, row0, lane, rows, m, ls);
  store_rows(lds + 8192 * wave, o, ls > 0.0f ? 1.0f / ls : 0.0f, lane, rows,
             [&](int r) { return a.out.p + (row0 + r) * a.out.sl + h * a.out.sh; });
}

// The pieces of a split item joined, in their order: a workgroup for 32 rows, a wave for 32 columns.
__global__ void __launch_bounds__(256) packed_fwd_join_kernel(const PackedArgs a) {
  const int lane = threadIdx.x & 63, db = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / PK_WAVES, wave = blockIdx.x % PK_WAVES;
  const PackedShare sh = {(int)(unit / (uint32_t)a.Hq), (int)(unit % (uint32_t)a.Hq), 0, true};
  int h, kv;
  pick_head(sh.head, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, sh.item);
  if (!item_fits(it, a.Tq, a.Tk)) return;
  const int pieces = pieces_of(a, sh, (it.bound + BN - 1) / BN);
  const int rows = it.rows - 32 * (int)wave;
  if (pieces == 1 || rows <= 0) return;
  const int row = 32 * wave + (lane & 31);
  float m = -INFINITY, l = 0.0f;
  for (int s = 0; s < pieces; ++s)
    m = fmaxf(m, part_of(a, sh, a.Hq, s, PK_PART_FWD)[PK_BLOCK * 128 + row]);
  floatx16 o;
  zero(o);
#pragma unroll 4
  for (int s = 0; s < pieces; ++s) {
    const float* part = part_of(a, sh, a.Hq, s, PK_PART_FWD);
    const float ms = part[PK_BLOCK * 128 + row];
    const float f = ms == -INFINITY ? 0.0f : fast_exp2((ms - m) * a.scale_log2);
    l += f * part[PK_BLOCK * 128 + PK_BLOCK + row];
    add_block(part, wave, db, lane, f, o);
  }
  const int64_t row0 = it.row0 + 32 * (int)wave;
  if (db == 0) store_lse(a, h, row0, lane, rows, m, l);
  store_block(o, l > 0.0f ? 1.0f / l : 0.0f, db, lane, rows,
              [&](int r) { return a.out.p + (row0 + r) * a.out.sl + h * a.out.sh; });
}

}  // namespace

hipError_t launch_packed_fwd(const PackedArgs& a, hipStream_t stream) {
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)packed_fwd_kernel, FWD_LDS, allowed);
  if (attr != hipSuccess) return attr;
  const uint32_t n = ((uint32_t)a.n_q_items + (uint32_t)a.n_split * (a.smax - 1)) * a.Hq;
  hipLaunchKernelGGL(packed_fwd_kernel, dim3(n), dim3(PK_WAVES * 64), FWD_LDS, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_split == 0) return e;
  hipLaunchKernelGGL(packed_fwd_join_kernel, dim3((uint32_t)a.n_split * a.Hq * PK_WAVES), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace lbw
