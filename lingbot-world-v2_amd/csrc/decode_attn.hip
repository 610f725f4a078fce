// Attention of one query token per sequence over its cache (gfx950).
//
//   out[b, h] = softmax(scale q[b, h] K^T) V over keys 0 .. len[b] - 1 of cache b, key/value head
//   h / (Hq / Hk); a sequence of no keys gives 0.
//
// Bound by reading K and V once. A workgroup takes one key/value head of one sequence (its query
// heads, up to 32, are the columns of S^T = K Q^T, so K and V are read once for the whole group)
// and one piece of the keys; its 4 waves take 32-key tiles in turn, each through an LDS ring of
// its own (two tiles of K and V, 32 KB), so no wave waits for another until the end, where the
// four results are joined. Pieces are joined by a second kernel in a fixed order.

#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int DW = 4;                       // waves per workgroup
constexpr int DT = 32;                      // keys per tile
constexpr int DT_B = DT * PK_ROWB;          // 8 KB
constexpr int STAGE_B = 2 * DT_B;           // K, then V
constexpr int RING_B = 2 * STAGE_B;         // per wave
constexpr int DEC_LDS = DW * RING_B;
constexpr int NCOPY = DT_B / 1024;          // copies per lane for K or V of a tile
constexpr int HEADS = 32;                   // query heads per workgroup

__global__ void __launch_bounds__(DW * 64, 1) decode_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  __shared__ float sm[DW][HEADS], sl[DW][HEADS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int group = a.Hq / a.Hk, blocks = (group + HEADS - 1) / HEADS;
  uint32_t id = blockIdx.x;
  const int kv = id % (uint32_t)a.Hk;
  id /= (uint32_t)a.Hk;
  const int hb = id % (uint32_t)blocks;
  id /= (uint32_t)blocks;
  const int split = id % (uint32_t)a.splits, b = id / (uint32_t)a.splits;
  const int h0 = kv * group + hb * HEADS;
  const int nh = min(HEADS, group - hb * HEADS);

  int len = a.lens[b];
  len = len < 0 ? 0 : (len > a.S ? a.S : len);
  len = __builtin_amdgcn_readfirstlane(len);
  const int tiles = (len + DT - 1) / DT;
  const int t0 = (int)((int64_t)tiles * split / a.splits) + wave;
  const int t1 = (int)((int64_t)tiles * (split + 1) / a.splits);

  u32x4 qf[8];
  load_rows(a.q.p + b * a.q.sl + h0 * a.q.sh, a.q.sh, nh, l32, hl, qf);
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(a.k + b * a.ksb + kv * a.ksh);
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(a.v + b * a.vsb + kv * a.vsh);

  const int ring = (int)lds_addr(lds) + RING_B * wave;
  const int ka = row_address(ring, l32, hl), va = tr_address(ring + DT_B, lane, hl);
  int crow[NCOPY], ccol[NCOPY];
#pragma unroll
  for (int i = 0; i < NCOPY; ++i) {
    crow[i] = 4 * i + (lane >> 4);
    ccol[i] = ((lane & 15) ^ swz(crow[i])) * 16;
  }
  auto issue = [&](int t, int stage) {
    const int64_t first = (int64_t)t * DT;
    const int last = len - 1 - t * DT;  // (rows past the end copy the last valid one)
    const unsigned char* kt = kb + first * a.ksl * 2;
    const unsigned char* vt = vb + first * a.vsl * 2;
    const uint32_t to = (uint32_t)ring + stage * STAGE_B;
#pragma unroll
    for (int i = 0; i < NCOPY; ++i) {
      const int r = crow[i] < last ? crow[i] : last;
      dma16_guarded(kt, (uint32_t)r * (uint32_t)(a.ksl * 2) + ccol[i], to + 1024 * i);
      dma16_guarded(vt, (uint32_t)r * (uint32_t)(a.vsl * 2) + ccol[i], to + DT_B + 1024 * i);
    }
  };

  floatx16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) zero(o[db]);
  float m = M_INIT, l = 0.0f;
  const float c = a.scale_log2;
  __builtin_amdgcn_s_waitcnt(0x0070);  // the query is there: only tile copies are counted below
  if (t0 < t1) issue(t0, 0);
  int stage = 0;
#pragma unroll 1
  for (int t = t0; t < t1; t += DW, stage ^= 1) {
    if (t + DW < t1) {
      issue(t + DW, stage ^ 1);
      static_assert(2 * NCOPY == 16, "the count below is a tile's copies");
      asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int at = stage * STAGE_B;
    floatx16 s;
    zero(s);
#pragma unroll
    for (int d = 0; d < 8; ++d) s = mfma32x32x16(read_row(ka, d, at), qf[d], s);
    const int left = len - (t * DT + 4 * hl);
    if (t * DT + DT > len) {
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
    // its reads of this stage are over before the next turn's copies into it
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  l = wave_sum_xor32(l);
  if (hl == 0) {
    sm[wave][l32] = l > 0.0f ? m : -INFINITY;
    sl[wave][l32] = l;
  }
  // O^T as rows [head][128] fp32 into the wave's ring (16 KB)
  float* mine = reinterpret_cast<float*>(lds + RING_B * wave);
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      floatx4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = o[db][4 * g + e];
      *reinterpret_cast<floatx4*>(mine + l32 * D + 32 * db + 8 * g + 4 * hl) = w;
    }
  __syncthreads();
  // thread: 4 values of one head at a time
  const int64_t BH = (int64_t)a.B * a.Hq;
  for (int x = threadIdx.x; x < nh * (D / 4); x += DW * 64) {
    const int hh = x / (D / 4), dq = 4 * (x % (D / 4));
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < DW; ++w) M = fmaxf(M, sm[w][hh]);
    float L = 0.0f;
    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < DW; ++w) {
      const float f = sm[w][hh] == -INFINITY ? 0.0f : fast_exp2((sm[w][hh] - M) * c);
      // (a wave without keys holds zeros)
      L += f * sl[w][hh];
      acc += f * *reinterpret_cast<const floatx4*>(
                     reinterpret_cast<const float*>(lds + RING_B * w) + hh * D + dq);
    }
    if (a.splits == 1) {
      const float inv = L > 0.0f ? 1.0f / L : 0.0f;
      u32x2 w;
      w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(a.out.p + b * a.out.sl + (h0 + hh) * a.out.sh + dq) = w;
    } else {
      const int64_t row = (int64_t)split * BH + (int64_t)b * a.Hq + h0 + hh;
      *reinterpret_cast<floatx4*>(a.part + row * D + dq) = acc;
      if (dq == 0) {
        float* st = a.part + (int64_t)a.splits * BH * D;
        st[row] = M;
        st[(int64_t)a.splits * BH + row] = L;
      }
    }
  }
}

// One wave per (sequence, query head): the pieces joined in their order.
__global__ void __launch_bounds__(256) decode_merge_kernel(const DecodeArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t BH = (int64_t)a.B * a.Hq, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= BH) return;
  const float* st = a.part + (int64_t)a.splits * BH * D;
  float M = -INFINITY;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, st[s * BH + row]);
  float L = 0.0f, x = 0.0f, y = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float ms = st[s * BH + row];
    const float f = ms == -INFINITY ? 0.0f : fast_exp2((ms - M) * a.scale_log2);
    L += f * st[(int64_t)a.splits * BH + s * BH + row];
    const float2 v = *reinterpret_cast<const float2*>(a.part + (s * BH + row) * D + 2 * lane);
    x += f * v.x;
    y += f * v.y;
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  const int b = (int)(row / a.Hq), h = (int)(row % a.Hq);
  *reinterpret_cast<uint32_t*>(a.out.p + b * a.out.sl + h * a.out.sh + 2 * lane) =
      pack_bf16x2(x * inv, y * inv);
}

}  // namespace

// Pieces of a sequence's keys: enough workgroups for every CU, pieces of 256 keys or more of the cache.
int decode_splits(int64_t B, int Hq, int Hk, int64_t S, int cus) {
  const int group = Hq / Hk;
  const int64_t units = B * Hk * ((group + HEADS - 1) / HEADS);
  int64_t s = (2 * cus + units - 1) / units;
  if (s > S / 256) s = S / 256;
  return (int)(s < 1 ? 1 : (s > 128 ? 128 : s));
}

hipError_t launch_decode(const DecodeArgs& a, hipStream_t stream) {
  static hipError_t attr = hipFuncSetAttribute((const void*)decode_kernel,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, DEC_LDS);
  if (attr != hipSuccess) return attr;
  const int group = a.Hq / a.Hk, blocks = (group + HEADS - 1) / HEADS;
  const int64_t n = (int64_t)a.B * a.splits * blocks * a.Hk;
  hipLaunchKernelGGL(decode_kernel, dim3((uint32_t)n), dim3(DW * 64), DEC_LDS, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = (int64_t)a.B * a.Hq;
  hipLaunchKernelGGL(decode_merge_kernel, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
