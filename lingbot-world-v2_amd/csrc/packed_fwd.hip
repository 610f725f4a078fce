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
#include "packed_loop.h"

namespace lbw {
namespace {

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
  TileCopy copy;
  copy.init(wave, lane);
  const uint32_t koff = copy.row_offset(ks), voff = copy.row_offset(vs);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;
  auto issue_k = [&](int u) { copy.issue(kb, ks, koff, (t0 + u) * BN, it.other_len, dst + (u & 1) * PK_TILE_B); };
  auto issue_v = [&](int u) {
    copy.issue(vb, vs, voff, (t0 + u) * BN, it.other_len, dst + V_AT + (u & 1) * PK_TILE_B);
  };

  floatx16 o[4];
  float m, l;
  attend_tiles(lds, wave, lane, qf, sreg(a.scale_log2), t0, T, Tw, lim, lim_lo, issue_k, issue_v, o, m, l);
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
