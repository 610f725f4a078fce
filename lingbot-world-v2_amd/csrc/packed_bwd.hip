// Gradient of attention over packed sequences (gfx950), from q, k, v, out, dout and lse.
//
//   P = exp(scale Q K^T - lse);  delta_i = sum_d dO O = sum_j P dP;  dS = P (dO V^T - delta)
//   dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO
//
// Two kernels, each with its sums in its own registers: no atomics, so the result does not depend
// on the order of workgroups. The first has 128 queries of a head per workgroup and walks their keys: it
// makes delta and dQ (three products a tile). The second has 128 keys of a key/value head and
// walks the queries of all heads of its group: dK and dV (four products a tile); its S starts from
// -lse / scale and its dP from -delta, so P and dS take one operation each from the accumulators.
// Both recompute S; P and dS go to bf16 as operands, one rounding each.
//
// Bound by matrix products and by what stands between them: 4680 + 3599 + 2340 causal tokens x 40/8 heads dQ 568 us
// (1091 TFLOP/s of its three products, MFMA busy 66 % of the cycles at 1.5 GHz), dK and dV 846 us (977 of its four,
// 58 % at 1.65 GHz; a library product of 16384^3 reaches 1364). The formula needs five products; S and dP are made in
// both kernels.

#include "capi_util.h"
#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int V_AT = 2 * PK_TILE_B;
constexpr int BWD_LDS = 4 * PK_TILE_B;
constexpr int STAT_AT = 4 * PK_TILE_B;             // -lse and delta of the query tiles, two stages
constexpr int DKV_GROUP_B = STAT_AT + 2 * 2 * BN * 4;  // LDS of a group of 4 waves

// ---- dQ: a lane holds one query's column of S^T = K Q^T and dP^T = V dO^T
__global__ void __launch_bounds__(PK_WAVES * 64, 2) packed_dq_kernel(const PackedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  int h, kv;
  const PackedShare sh = pick_share(a, blockIdx.x, a.Hq);
  pick_head(sh.head, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, sh.item);
  if (!item_fits(it, a.Tq, a.Tk)) return;
  const int n_tiles = (it.bound + BN - 1) / BN, pieces = pieces_of(a, sh, n_tiles);
  if (sh.piece >= pieces) return;
  const int t0 = (int)((int64_t)n_tiles * sh.piece / pieces);
  const int T = (int)((int64_t)n_tiles * (sh.piece + 1) / pieces);
  const int r0 = 32 * wave, rows = it.rows - r0;
  const bool active = rows > 0;

  u32x4 qf[8], gf[8];
  float nlse2 = -INFINITY, delta = 0.0f;  // -lse log2(e); no key seen (lse = -inf): every p becomes 0
  if (active) {
    const int64_t row = it.row0 + r0;
    load_rows(a.q.p + row * a.q.sl + h * a.q.sh, a.q.sl, rows, l32, hl, qf);
    load_rows(a.dout.p + row * a.dout.sl + h * a.dout.sh, a.dout.sl, rows, l32, hl, gf);
    const float x = l32 < rows ? a.lse[(int64_t)h * a.Tq + row + l32] : -INFINITY;
    nlse2 = x == -INFINITY ? -INFINITY : -x * LOG2E;
    u32x4 of[8];
    load_rows(a.o.p + row * a.o.sl + h * a.o.sh, a.o.sl, rows, l32, hl, of);
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        delta += bf16_lo(gf[s][w]) * bf16_lo(of[s][w]) + bf16_hi(gf[s][w]) * bf16_hi(of[s][w]);
    delta = wave_sum_xor32(delta);
  }
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(
      a.k.p + (int64_t)it.other0 * a.k.sl + kv * a.k.sh);
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(
      a.v.p + (int64_t)it.other0 * a.v.sl + kv * a.v.sh);
  const int64_t ks = a.k.sl * 2, vs = a.v.sl * 2;
  const int i0 = it.pos0 + r0;
  auto limit = [&](int i) {
    const int64_t x = (int64_t)i + it.shift + 1;
    return (int)(x < 0 ? 0 : (x < it.other_len ? x : it.other_len));
  };
  const int lim = limit(i0 + l32);
  const int lim_lo = limit(i0), lim_hi = limit(i0 + (rows < 32 ? rows : 32) - 1);

  const int lds0 = (int)lds_addr(lds);
  const int ra0 = row_address(lds0, l32, hl), ta0 = tr_address(lds0, lane, hl);
  TileCopy copy;
  copy.init(wave, lane);
  const uint32_t koff = copy.row_offset(ks), voff = copy.row_offset(vs);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;
  const float c = a.scale_log2;
  // Out is rounded, and where a row sees few keys its error, in delta, is as large as all others together
  // (dQ's error at sequences of 5 to 512 tokens: 1.65 roundings of the result; with delta exact up to 256
  // keys 1.41, what the roundings of dS and dQ themselves give). So an item of few tiles goes over them
  // first for delta = sum_j P dP in 32 bits: 2 to 3 % of the gradient at 512 tokens, nothing at 4680.
  const bool exact = n_tiles <= 4 && pieces == 1;
  if (exact) {
    delta = 0.0f;
#pragma unroll 1
    for (int u = 0; u < T; ++u) {
      barrier_nofence();  // everybody is past the tile before
      copy.issue(kb, ks, koff, u * BN, it.other_len, dst);
      copy.issue(vb, vs, voff, u * BN, it.other_len, dst + V_AT);
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
      barrier_nofence();
      if (!active || u * BN >= lim_hi) continue;
#pragma unroll 1
      for (int at = 0; at < 2; ++at) {
        const int ra = opaque(ra0 + at * 32 * PK_ROWB);
        floatx16 s, d;
        zero(s);
        zero(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s = mfma32x32x16(read_row(ra, i, 0), qf[i], s);
          d = mfma32x32x16(read_row(ra, i, V_AT), gf[i], d);
        }
        const int left = lim - (u * BN + 32 * at + 4 * hl);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          delta += acc_row(r) < left ? fast_exp2(__builtin_fmaf(s[r], c, nlse2)) * d[r] : 0.0f;
      }
      // (its reads are over before the next barrier)
      __builtin_amdgcn_s_waitcnt(0x0070);
    }
    delta = wave_sum_xor32(delta);
    barrier_nofence();
  }
  floatx16 acc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(acc[db]);
  if (t0 < T) {
    copy.issue(kb, ks, koff, t0 * BN, it.other_len, dst + (t0 & 1) * PK_TILE_B);
    copy.issue(vb, vs, voff, t0 * BN, it.other_len, dst + V_AT + (t0 & 1) * PK_TILE_B);
  }
#pragma unroll 1
  for (int u = t0; u < T; ++u) {
    const int st = (u & 1) * PK_TILE_B;
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    barrier_nofence();
    if (u + 1 < T) {
      copy.issue(kb, ks, koff, (u + 1) * BN, it.other_len, dst + (PK_TILE_B - st));
      copy.issue(vb, vs, voff, (u + 1) * BN, it.other_len, dst + V_AT + (PK_TILE_B - st));
    }
    if (!active || u * BN >= lim_hi) continue;
    // The tile's two 32-key blocks: S0; dP0 beside exp(S0); S1 beside dS0; dQ's product with dS0 and dP1
    // beside exp(S1); dS1; dQ's product with dS1. Fragments two products ahead.
    const int ra = ra0 + st, ta = ta0 + st;
    constexpr int B1 = 32 * PK_ROWB;
    floatx16 s0, s1, dp;
    u32x4 f[4], df[2];
    auto mask = [&](floatx16& s, int key0) {
      if (key0 + 32 > lim_lo) {
        const int left = lim - (key0 + 4 * hl);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = acc_row(r) < left ? s[r] : -INFINITY;
      }
    };
    auto exps = [&](floatx16& s, int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) s[2 * i + e] = fast_exp2(__builtin_fmaf(s[2 * i + e], c, nlse2));
    };
    auto grad = [&](const floatx16& p, int i) {
      df[i >> 2][i & 3] = pack_bf16x2(p[2 * i] * (dp[2 * i] - delta), p[2 * i + 1] * (dp[2 * i + 1] - delta));
    };
    zero(s0);
    f[0] = read_row(ra, 0, 0);
    f[1] = read_row(ra, 1, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[(i + 2) & 3] = i + 2 < 8 ? read_row(ra, i + 2, 0) : read_row(ra, i - 6, V_AT);
      s0 = mfma32x32x16(f[i & 3], qf[i], s0);
      __builtin_amdgcn_sched_barrier(0);
    }
    mask(s0, u * BN);
    zero(dp);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[(i + 2) & 3] = i + 2 < 8 ? read_row(ra, i + 2, V_AT) : read_row(ra, i - 6, B1);
      dp = mfma32x32x16(f[i & 3], gf[i], dp);
      exps(s0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" : "+v"(s0));  // (the exponentials stay here, not sunk to their use past a branch)
    zero(s1);
    u32x4 g[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + 2 < 8) f[(i + 2) & 3] = read_row(ra, i + 2, B1);
      else g[i - 6] = read_tr(ta, i - 6, 0, 0);
      s1 = mfma32x32x16(f[i & 3], qf[i], s1);
      grad(s0, i);
      if (i >= 6) f[(i + 2) & 3] = read_row(ra, i - 6, B1 + V_AT);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" : "+v"(df[0]), "+v"(df[1]));
    mask(s1, u * BN + 32);
    zero(dp);
    // (fragment i of dQ's product: d-block i % 4, k-half i / 4)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + 2 < 8) f[(i + 2) & 3] = read_row(ra, i + 2, B1 + V_AT);
      g[(i + 2) & 3] = i + 2 < 8 ? read_tr(ta, (i + 2) & 3, (i + 2) >> 2, 0) : read_tr(ta, i - 6, 0, B1);
      dp = mfma32x32x16(f[i & 3], gf[i], dp);
      acc[i & 3] = mfma32x32x16(g[i & 3], df[i >> 2], acc[i & 3]);
      exps(s1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) grad(s1, i);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + 2 < 8) g[(i + 2) & 3] = read_tr(ta, (i + 2) & 3, (i + 2) >> 2, B1);
      acc[i & 3] = mfma32x32x16(g[i & 3], df[i >> 2], acc[i & 3]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();
  if (!active) return;
  if (hl == 0 && sh.piece == 0 && l32 < rows) {  // for the other kernel
    const int64_t at = (int64_t)h * a.Tq + it.row0 + r0 + l32;
    a.ndelta[at] = -delta;
    a.nlse[at] = nlse2 == -INFINITY ? -INFINITY : nlse2 / c;
  }
  if (pieces > 1) {
    store_acc(part_of(a, sh, a.Hq, sh.piece, PK_PART_DQ), wave, lane, acc);
    return;
  }
  store_rows(lds + 8192 * wave, acc, a.scale, lane, rows, [&](int r) {
    return a.dq.p + (int64_t)(it.row0 + r0 + r) * a.dq.sl + h * a.dq.sh;
  });
}

// The pieces of a split query item added up, in their order: a workgroup for 32 rows, a wave for 32 columns.
__global__ void __launch_bounds__(256) packed_dq_join_kernel(const PackedArgs a) {
  const int lane = threadIdx.x & 63, db = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / PK_WAVES, wave = blockIdx.x % PK_WAVES;
  const PackedShare sh = {(int)(unit / (uint32_t)a.Hq), (int)(unit % (uint32_t)a.Hq), 0, true};
  int h, kv;
  pick_head(sh.head, a.Hk, a.Hq / a.Hk, h, kv);
  const PackedItem it = load_item(a.q_items, sh.item);
  if (!item_fits(it, a.Tq, a.Tk)) return;
  const int pieces = pieces_of(a, sh, (it.bound + BN - 1) / BN), rows = it.rows - 32 * (int)wave;
  if (pieces == 1 || rows <= 0) return;
  floatx16 acc;
  zero(acc);
#pragma unroll 4
  for (int s = 0; s < pieces; ++s) add_block(part_of(a, sh, a.Hq, s, PK_PART_DQ), wave, db, lane, 1.0f, acc);
  store_block(acc, a.scale, db, lane, rows, [&](int r) {
    return a.dq.p + (int64_t)(it.row0 + 32 * (int)wave + r) * a.dq.sl + h * a.dq.sh;
  });
}

// ---- dK, dV: a lane holds one key's column of S = Q K^T and dP = dO V^T
// 192 of a wave's 256 registers hold dK, dV, K and V; S, dP and the fragments take 50 more. So nothing that
// can be had again in a few instructions is kept across the loop: the lane index and what follows from it.
__device__ __forceinline__ int lane_now() {
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (uint32_t)opaque(0)));
}
constexpr int GROUPS = 2;  // wave groups of a workgroup, each with its share of an item's query tiles
constexpr int FRAG_AT = GROUPS * DKV_GROUP_B;    // each wave's last fragment of K and of V: 2 KB
constexpr int DKV_LDS = FRAG_AT + GROUPS * PK_WAVES * 2048;
// Where there are few items a workgroup takes HALF of one, 64 keys: two waves of a group share a block of 32
// keys, each with every second block of 32 queries (12 tiles of 3 heads 43 to 30 us).
template <bool HALF>
__global__ void __launch_bounds__(GROUPS * PK_WAVES * 64, 1) packed_dkv_kernel(const PackedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_id % PK_WAVES, grp = wave_id / PK_WAVES;
  const int hl = lane >> 5, l32 = lane & 31;
  const PackedShare sh = pick_share(a, HALF ? blockIdx.x >> 1 : blockIdx.x, a.Hk);
  const int kv = sh.head, group = a.Hq / a.Hk;
  const PackedItem it = load_item(a.k_items, sh.item);
  if (!item_fits(it, a.Tk, a.Tq)) return;
  // query tiles of a head, and of the group's heads one after another; this piece's, this group's
  const int t_first = it.bound / BN, t_end = (it.other_len + BN - 1) / BN;
  const int per = it.bound < it.other_len ? t_end - t_first : 0;
  const int all = per * group, pieces = pieces_of(a, sh, all);
  if (sh.piece >= pieces) return;
  const int p0 = (int)((int64_t)all * sh.piece / pieces);
  const int mine = (int)((int64_t)all * (sh.piece + 1) / pieces) - p0;
  const int n0 = p0 + mine * grp / GROUPS, T = p0 + mine * (grp + 1) / GROUPS;
  const int Tmax = n0 + (mine + GROUPS - 1) / GROUPS;  // the loop's end, the same count in both groups
  const int part0 = HALF ? 64 * (int)(blockIdx.x & 1) : 0;
  if (HALF && it.rows <= part0) return;
  const int r0 = part0 + 32 * (HALF ? wave & 1 : wave), rows = it.rows - r0;
  const bool active = rows > 0;

  u32x4 kf[8], vf[8];
  if (active) {
    const int64_t row = it.row0 + r0;
    load_rows(a.k.p + row * a.k.sl + kv * a.k.sh, a.k.sl, rows, l32, hl, kf);
    load_rows(a.v.p + row * a.v.sl + kv * a.v.sh, a.v.sl, rows, l32, hl, vf);
  }
  // the eighth fragments wait in LDS rather than in registers
  const int frag = (int)lds_addr(lds) + FRAG_AT + 2048 * wave_id;
  {
    unsigned char* const d = lds + FRAG_AT + 2048 * wave_id + 16 * lane;
    *reinterpret_cast<u32x4*>(d) = kf[7];
    *reinterpret_cast<u32x4*>(d + 1024) = vf[7];
    wave_lds_fence();
  }
  // first query that sees this lane's key, and the wave's smallest and largest such
  const int j0 = it.pos0 + r0;
  auto first = [&](int j) {
    const int64_t x = (int64_t)j - it.shift;
    return (int)(x < 0 ? 0 : (x < it.other_len ? x : it.other_len));
  };
  const int lo_min = first(j0), lo_max = first(j0 + 31);

  const int lds0 = (int)lds_addr(lds) + DKV_GROUP_B * grp;
  const int ra0 = row_address(lds0, l32, hl), ta0 = tr_address(lds0, lane, hl);
  const uint32_t dst = (uint32_t)lds0 + 1024 * PK_NDMA * wave;
  floatx16 dk[4], dv[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    zero(dk[db]);
    zero(dv[db]);
  }
  const float c = a.scale_log2;
  const int64_t qs = a.q.sl * 2, gs = a.dout.sl * 2;
  // The next query tile to fetch: head and tile of it, stepped along (no division per tile).
  int nh = kv * group + (per > 0 ? n0 / per : 0), nt = t_first + (per > 0 ? n0 % per : 0);
  // query tile n into stage n % 2; waves 0 and 1 fetch its rows' -lse / scale and -delta (rows past the
  // sequence's end: the last one's)
  auto issue = [&](int n) {
    const int first_row = nt * BN, ln = lane_now();
    TileCopy copy;
    copy.init(wave, ln);
    const uint32_t qoff = copy.row_offset(qs), goff = copy.row_offset(gs);
    const uint32_t to = dst + (n & 1) * PK_TILE_B;
    if (wave < 2) {
      const int r = min(first_row + ln, it.other_len - 1);
      const float* x = (wave == 0 ? a.nlse : a.ndelta) + (int64_t)nh * a.Tq + it.other0 + r;
      dma4((uint64_t)(uintptr_t)x, (uint32_t)lds0 + STAT_AT + ((n & 1) * 2 + wave) * BN * 4);
    }
    copy.issue(reinterpret_cast<const unsigned char*>(a.q.p + (int64_t)it.other0 * a.q.sl + nh * a.q.sh),
               qs, qoff, first_row, it.other_len, to);
    copy.issue(reinterpret_cast<const unsigned char*>(a.dout.p + (int64_t)it.other0 * a.dout.sl +
                                                      nh * a.dout.sh),
               gs, goff, first_row, it.other_len, to + V_AT);
    if (++nt == t_end) {
      nt = t_first;
      ++nh;
    }
  };
  int ct = nt;  // the tile being worked on
  if (n0 < T) issue(n0);
#pragma unroll 1
  for (int n = n0; n < Tmax; ++n) {
    const int st = (n & 1) * PK_TILE_B;
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    barrier_nofence();
    if (n + 1 < T) issue(n + 1);
    const int row0 = ct * BN;
    ct = ct + 1 == t_end ? t_first : ct + 1;
    if (!active || n >= T || row0 + BN <= lo_min) continue;
#pragma unroll 1
    for (int qb = HALF ? wave >> 1 : 0; qb < (HALF ? (wave >> 1) + 1 : 2); ++qb) {
      // (each product's fragment addresses are taken anew: kept for two of them, they spill others)
      const int ra = opaque(ra0 + st + qb * 32 * PK_ROWB);
      const int sa = lds0 + STAT_AT + (n & 1) * 2 * BN * 4 + 128 * qb + 16 * (lane_now() >> 5);
      // S (from -lse / scale on), then dP (from -delta on) beside the exponentials, then dV beside dS, then
      // dK: fragments two products ahead
      floatx16 s, dp;
      auto start = [&](floatx16& x, int at) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const u32x4 v = lds_read_b128(sa + 32 * g + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * g + e] = __uint_as_float(v[e]);
        }
      };
      start(s, 0);
      u32x4 f[3];
      const int fa = frag + 16 * lane_now();
      u32x4 last = lds_read_b128(fa);
      f[0] = read_row(ra, 0, 0);
      f[1] = read_row(ra, 1, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[(i + 2) % 3] = i + 2 < 8 ? read_row(ra, i + 2, 0) : read_row(ra, i - 6, V_AT);
        s = mfma32x32x16(f[i % 3], i < 7 ? kf[i] : last, s);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int i0 = row0 + 32 * qb;
      if (i0 < lo_max || i0 + 32 > it.other_len) {  // (register r is query i0 + 4 hl + acc_row(r))
        const int ln = lane_now(), q0 = i0 + 4 * (ln >> 5);
        const int skip = first(j0 + (ln & 31)) - q0, end = it.other_len - q0;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = acc_row(r) >= skip && acc_row(r) < end ? s[r] : -INFINITY;
      }
      // (fragment i of the 8 + 8 + 8 products from here on is in f[(i + 2) % 3])
      const int rb = opaque(ra), ta = opaque(ta0 + st + qb * 32 * PK_ROWB);
      u32x4 pf[2], df[2];
      start(dp, BN * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[(i + 4) % 3] = i + 2 < 8 ? read_row(rb, i + 2, V_AT) : read_tr(ta, i - 6, 0, V_AT);
        if (i == 4) last = lds_read_b128(fa + 1024);
        dp = mfma32x32x16(f[(i + 2) % 3], i < 7 ? vf[i] : last, dp);
#pragma unroll
        for (int e = 0; e < 2; ++e) s[2 * i + e] = fast_exp2(s[2 * i + e] * c);
        if (i < 4) pf[0][i] = pack_bf16x2(s[2 * i], s[2 * i + 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // products 8 .. 15: dV, k-half (i / 4) % 2, d-block i % 4; 16 .. 23: dK
      const int tb = opaque(ta);
#pragma unroll
      for (int i = 8; i < 16; ++i) {
        const int n = i + 2;
        f[(i + 4) % 3] = read_tr(n < 16 ? ta : tb, n & 3, (n >> 2) & 1, n < 16 ? V_AT : 0);
        dv[i & 3] = mfma32x32x16(f[(i + 2) % 3], pf[(i >> 2) & 1], dv[i & 3]);
        const int w = i - 8;  // word w / 4, w % 4 of the operands
        if (w < 4) pf[1][w] = pack_bf16x2(s[8 + 2 * w], s[8 + 2 * w + 1]);
        df[w >> 2][w & 3] = pack_bf16x2(s[2 * w] * dp[2 * w], s[2 * w + 1] * dp[2 * w + 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 16; i < 24; ++i) {
        const int n = i + 2;
        if (n < 24) f[(i + 4) % 3] = read_tr(tb, n & 3, (n >> 2) & 1, 0);
        dk[i & 3] = mfma32x32x16(f[(i + 2) % 3], df[(i >> 2) & 1], dk[i & 3]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrier_nofence();
  {
    // Group 1 hands its sums over in register order, 16 bytes per lane: dK through its own LDS, dV
    // through group 0's. Then, where two waves share keys, the second of group 0 does.
    unsigned char* const g1 = lds + DKV_GROUP_B;
    const int ln = lane_now();
    auto give = [&]() {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const floatx16 &y = dk[x >> 2], &z = dv[x >> 2];
        const int e = 4 * (x & 3), at = 16384 * wave + 1024 * x + 16 * ln;
        *reinterpret_cast<floatx4*>(g1 + at) = floatx4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        *reinterpret_cast<floatx4*>(lds + at) = floatx4{z[e], z[e + 1], z[e + 2], z[e + 3]};
      }
    };
    auto take = [&](int from) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int at = 16384 * from + 1024 * x + 16 * ln;
        const floatx4 y = *reinterpret_cast<const floatx4*>(g1 + at);
        const floatx4 z = *reinterpret_cast<const floatx4*>(lds + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dk[x >> 2][4 * (x & 3) + e] += y[e];
          dv[x >> 2][4 * (x & 3) + e] += z[e];
        }
      }
    };
    if (grp == 1) give();
    __syncthreads();
    if (grp == 0) take(wave);
    __syncthreads();  // the sums are read: the LDS is free again
    if constexpr (HALF) {
      if (grp == 0 && wave >= 2) give();
      __syncthreads();
      if (grp == 0 && wave < 2) take(wave + 2);
      __syncthreads();
      if (wave >= 2) return;
    }
    if (grp == 1) return;
  }
  if (!active) return;
  if (pieces > 1) {
    const int ln1 = lane_now(), slot = part0 / 32 + wave;
    float* const part = part_of(a, sh, a.Hk, sh.piece, PK_PART_DKV);
    store_acc(part, slot, ln1, dk);
    store_acc(part + PK_BLOCK * 128, slot, ln1, dv);
    return;
  }
  const int ln = lane_now();
  store_rows(lds + 8192 * wave, dk, a.scale, ln, rows, [&](int r) {
    return a.dk.p + (int64_t)(it.row0 + r0 + r) * a.dk.sl + kv * a.dk.sh;
  });
  wave_lds_fence();
  store_rows(lds + 8192 * wave, dv, 1.0f, ln, rows, [&](int r) {
    return a.dv.p + (int64_t)(it.row0 + r0 + r) * a.dv.sl + kv * a.dv.sh;
  });
}

// The pieces of a split key item added up, in their order: a workgroup for 32 rows of dK or dV.
__global__ void __launch_bounds__(256) packed_dkv_join_kernel(const PackedArgs a) {
  const int lane = threadIdx.x & 63, db = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / (2 * PK_WAVES), which = blockIdx.x / PK_WAVES % 2, wave = blockIdx.x % PK_WAVES;
  const PackedShare sh = {(int)(unit / (uint32_t)a.Hk), (int)(unit % (uint32_t)a.Hk), 0, true};
  const PackedItem it = load_item(a.k_items, sh.item);
  if (!item_fits(it, a.Tk, a.Tq)) return;
  const int per = it.bound < it.other_len ? (it.other_len + BN - 1) / BN - it.bound / BN : 0;
  const int pieces = pieces_of(a, sh, per * (a.Hq / a.Hk)), rows = it.rows - 32 * (int)wave;
  if (pieces == 1 || rows <= 0) return;
  floatx16 acc;
  zero(acc);
#pragma unroll 4
  for (int s = 0; s < pieces; ++s)
    add_block(part_of(a, sh, a.Hk, s, PK_PART_DKV) + which * PK_BLOCK * 128, wave, db, lane, 1.0f, acc);
  const RowsOut out = which == 0 ? a.dk : a.dv;
  store_block(acc, which == 0 ? a.scale : 1.0f, db, lane, rows, [&](int r) {
    return out.p + (int64_t)(it.row0 + 32 * (int)wave + r) * out.sl + sh.head * out.sh;
  });
}

}  // namespace

hipError_t launch_packed_dq(const PackedArgs& a, hipStream_t stream) {
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)packed_dq_kernel, BWD_LDS, allowed);
  if (attr != hipSuccess) return attr;
  const uint32_t n = ((uint32_t)a.n_q_items + (uint32_t)a.n_split * (a.smax - 1)) * a.Hq;
  hipLaunchKernelGGL(packed_dq_kernel, dim3(n), dim3(PK_WAVES * 64), BWD_LDS, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_split == 0) return e;
  hipLaunchKernelGGL(packed_dq_join_kernel, dim3((uint32_t)a.n_split * a.Hq * PK_WAVES), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

namespace {
template <bool HALF>
hipError_t run_dkv(const PackedArgs& a, uint32_t n, hipStream_t stream) {
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)packed_dkv_kernel<HALF>, DKV_LDS, allowed);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL(packed_dkv_kernel<HALF>, dim3(n), dim3(GROUPS * PK_WAVES * 64), DKV_LDS, stream, a);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_packed_dkv(const PackedArgs& a, hipStream_t stream) {
  const uint32_t n = ((uint32_t)a.n_k_items + (uint32_t)a.n_split * (a.smax - 1)) * a.Hk;
  const hipError_t e = a.halves ? run_dkv<true>(a, 2 * n, stream) : run_dkv<false>(a, n, stream);
  if (e != hipSuccess || a.n_split == 0) return e;
  hipLaunchKernelGGL(packed_dkv_join_kernel, dim3((uint32_t)a.n_split * a.Hk * 2 * PK_WAVES), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace lbw
