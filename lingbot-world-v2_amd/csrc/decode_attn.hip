// Attention of one query token per sequence over its cache (gfx950).
//
//   out[b, h] = softmax(scale q[b, h] K^T) V over keys 0 .. len[b] - 1 of cache b, key/value head
//   h / (Hq / Hk); a sequence of no keys gives 0.
//
// Bound by reading K and V once. A workgroup works for one key/value head: its query heads, up to 32,
// are the columns of S^T = K Q^T, so K and V are read once for the whole group. Its 4 or 8 waves take 32-key
// tiles in turn, each through 16 KB of LDS of its own (a tile of K, one of V: the next tile's K is
// fetched while this one's V is worked on, and the other way round), so no wave waits for another until a
// sequence ends, where their results are joined; two workgroups of 4 share a CU.
//
// Either a workgroup has one whole sequence, or (few sequences, long caches) the keys of the whole batch,
// laid end to end, are cut into equal pieces, as many as workgroups run at once: lengths are known on the
// device only, and ragged ones then cost no time. A piece may end inside a sequence; what
// belongs to one sequence is joined by a second kernel, in order.
//
// Eight sequences of 240000 keys together x 40/8 heads (0.98 GB) 171 us, 5.7 TB/s, and 5.4 us for the join;
// one of 500 keys 7.4 us, a whole sequence per workgroup.

#include <algorithm>

#include "capi_util.h"
#include "packed_tiles.h"

namespace lbw {
namespace {

constexpr int DT = 32;                      // keys per tile
constexpr int DT_B = DT * PK_ROWB;          // 8 KB
constexpr int RING_B = 2 * DT_B;            // per wave: K, V
constexpr int NCOPY = DT_B / 1024;          // copies per lane for K or V of a tile
constexpr int HEADS = 32;                   // query heads per workgroup

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ int64_t scalar64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int tiles_of(const DecodeArgs& a, int b) {
  const int n = a.lens[b];
  return ((n < 0 ? 0 : (n > a.S ? a.S : n)) + DT - 1) / DT;
}
// Tiles of all sequences together and, with `upto`, of those before it.
__device__ __forceinline__ void count_tiles_of(const DecodeArgs& a, int lane, int upto, int64_t& all,
                                               int64_t& before) {
  int64_t x = 0, y = 0;
  for (int b = lane; b < a.B; b += 64) {
    const int n = tiles_of(a, b);
    x += n;
    if (b < upto) y += n;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    x += __shfl_xor(x, o);
    y += __shfl_xor(y, o);
  }
  all = scalar64(x);
  before = scalar64(y);
}
// The sequence that tile `t` belongs to (0 <= t < all), and the tiles before it.
__device__ __forceinline__ int find_sequence(const DecodeArgs& a, int lane, int64_t t, int64_t& before) {
  int64_t base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? tiles_of(a, b0 + lane) : 0;
    int64_t sum = n;  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t y = __shfl_up(sum, o);
      if (lane >= o) sum += y;
    }
    const uint64_t past = __ballot(base + sum > t);
    if (past != 0) {
      const int l = __ffsll((unsigned long long)past) - 1;
      before = scalar64(base + __shfl(sum - n, l));
      return __builtin_amdgcn_readfirstlane(b0 + l);
    }
    base += __shfl(sum, 63);
  }
  before = base;
  return a.B;
}

template <int DW>  // waves per workgroup
__global__ void __launch_bounds__(DW * 64, 2) decode_kernel(const DecodeArgs a) {
  constexpr int DEC_LDS = DW * RING_B;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int group = a.Hq / a.Hk, blocks = (group + HEADS - 1) / HEADS;
  uint32_t id = blockIdx.x;
  const int kv = id % (uint32_t)a.Hk;
  id /= (uint32_t)a.Hk;
  const int hb = id % (uint32_t)blocks, piece = id / (uint32_t)blocks;
  const int h0 = kv * group + hb * HEADS;
  const int nh = min(HEADS, group - hb * HEADS);

  // this workgroup's tiles [at, end) of the batch laid end to end, from sequence b on
  int b = piece;
  int64_t at = 0, end = 1, before = 0;
  if (a.pieces > 0) {
    int64_t all, none;
    count_tiles_of(a, lane, 0, all, none);
    // (no more pieces than tiles: an empty one between two parts of a sequence would leave a row unwritten)
    const int64_t pieces = all < a.pieces ? all : a.pieces;
    if (piece >= pieces) return;
    at = all * piece / pieces;
    end = all * (piece + 1) / pieces;
    b = find_sequence(a, lane, at, before);
    if (b >= a.B) return;
  }

  const int ring = (int)lds_addr(lds) + RING_B * wave;
  const int ka = row_address(ring, l32, hl), va = tr_address(ring + DT_B, lane, hl);
  // copy i of a tile: rows 4 i + lane / 16, chunk (lane % 16) ^ swz(row); rows i and i + 4 share the chunk
  const int crow = lane >> 4, ccol = ((lane & 15) ^ swz(lane >> 4)) * 16;
  const uint32_t koff = (uint32_t)crow * (uint32_t)(a.ksl * 2), voff = (uint32_t)crow * (uint32_t)(a.vsl * 2);
  const float c = sreg(a.scale_log2);

  do {
    int len = a.lens[b];
    len = __builtin_amdgcn_readfirstlane(len < 0 ? 0 : (len > a.S ? a.S : len));
    const int tiles = (len + DT - 1) / DT;
    // this sequence's tiles of the piece (without pieces: all of them)
    const int s0 = a.pieces > 0 ? (int)(at - before) : 0;
    const int s1 = a.pieces > 0 ? (int)(end - before < tiles ? end - before : tiles) : tiles;

    u32x4 qf[8];
    load_rows(a.q.p + b * a.q.sl + h0 * a.q.sh, a.q.sh, nh, l32, hl, qf);
    const unsigned char* kb = reinterpret_cast<const unsigned char*>(a.k + b * a.ksb + kv * a.ksh);
    const unsigned char* vb = reinterpret_cast<const unsigned char*>(a.v + b * a.vsb + kv * a.vsh);
    auto issue = [&](const unsigned char* base, int64_t stride_b, uint32_t off, int t, uint32_t to) {
      // (scalar: what the compiler cannot see is the same in every lane)
      const unsigned char* p = reinterpret_cast<const unsigned char*>(
          (uintptr_t)scalar64((int64_t)(uintptr_t)(base + (int64_t)t * DT * stride_b)));
      const int last = len - 1 - t * DT;
      if (last >= DT - 1) {
#pragma unroll
        for (int i = 0; i < NCOPY; ++i)
          dma16_guarded(p + 4 * i * stride_b, off + (ccol ^ ((i & 3) << 4)), to + 1024 * i);
      } else {  // (rows past the end copy the last one)
#pragma unroll
        for (int i = 0; i < NCOPY; ++i) {
          const int r = crow + 4 * i < last ? crow + 4 * i : last;
          dma16_guarded(p, (uint32_t)r * (uint32_t)stride_b + (ccol ^ ((i & 3) << 4)), to + 1024 * i);
        }
      }
    };
    auto issue_k = [&](int t) { issue(kb, a.ksl * 2, koff, t, (uint32_t)ring); };
    auto issue_v = [&](int t) { issue(vb, a.vsl * 2, voff, t, (uint32_t)ring + DT_B); };
    static_assert(NCOPY == 8, "the counts below are a tile's copies");

    floatx16 o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db) zero(o[db]);
    float m = M_INIT, l = 0.0f;
    __builtin_amdgcn_s_waitcnt(0x0070);  // the query is there: only tile copies are counted below
    int t = s0 + wave;
    if (t < s1) {
      issue_k(t);
      issue_v(t);
    }
#pragma unroll 1
    for (; t < s1; t += DW) {
      const bool more = t + DW < s1;
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // K is there (V may be on its way)
      floatx16 s;
      zero(s);
#pragma unroll
      for (int d = 0; d < 8; ++d) s = mfma32x32x16(read_row(ka, d, 0), qf[d], s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its reads are over before K is overwritten
      if (more) issue_k(t + DW);
      if (t * DT + DT > len) {
        const int left = len - (t * DT + 4 * hl);
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
      if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // V is there (the next K may not be)
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int mm = 0; mm < 2; ++mm) o[db] = mfma32x32x16(read_tr(va, db, mm, 0), pf[mm], o[db]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) issue_v(t + DW);
    }
    l = wave_sum_xor32(l);
    // O^T as rows [head][128] fp32 into the wave's LDS, m and l behind the rings
    float* const sm = reinterpret_cast<float*>(lds + DEC_LDS);
    float* const sl = sm + DW * HEADS;
    if (hl == 0) {  // (no keys: a reference of -inf, weight 0; a sum that is NaN keeps its own and stays)
      sm[wave * HEADS + l32] = l == 0.0f ? -INFINITY : m;
      sl[wave * HEADS + l32] = l;
    }
    float* mine = reinterpret_cast<float*>(lds + RING_B * wave);
    if (l32 < nh) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          floatx4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = o[db][4 * g + e];
          *reinterpret_cast<floatx4*>(mine + l32 * D + 32 * db + 8 * g + 4 * hl) = w;
        }
    }
    __syncthreads();
    const bool whole = s1 - s0 == tiles;
    for (int x = threadIdx.x; x < nh * (D / 4); x += DW * 64) {  // 4 values of one head at a time
      const int hh = x / (D / 4), dq = 4 * (x % (D / 4));
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < DW; ++w) M = fmaxf(M, sm[w * HEADS + hh]);
      float L = 0.0f;
      floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < DW; ++w) {
        const float mw = sm[w * HEADS + hh], f = mw == -INFINITY ? 0.0f : fast_exp2((mw - M) * c);
        // (a wave without keys holds zeros)
        L += f * sl[w * HEADS + hh];
        acc += f * *reinterpret_cast<const floatx4*>(
                       reinterpret_cast<const float*>(lds + RING_B * w) + hh * D + dq);
      }
      if (whole) {
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        u32x2 w;
        w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
        w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<u32x2*>(a.out.p + b * a.out.sl + (h0 + hh) * a.out.sh + dq) = w;
      } else {
        // (piece + b: the parts of a head in the order of their keys, each in a row of its own, as the
        // next part has another piece or a later sequence, or both)
        const int64_t rows = (int64_t)a.pieces + a.B, row = (h0 + hh) * rows + piece + b;
        *reinterpret_cast<floatx4*>(a.part + row * D + dq) = acc;
        if (dq == 0) {
          float* st = a.part + a.Hq * rows * D;
          st[row] = M;
          st[a.Hq * rows + row] = L;
        }
      }
    }
    if (a.pieces == 0) return;
    at = before + tiles;
    if (at >= end) return;
    // the next sequence with keys
    before = at;
    do {
      b = __builtin_amdgcn_readfirstlane(b + 1);
    } while (b < a.B && __builtin_amdgcn_readfirstlane(tiles_of(a, b)) == 0);
    if (b >= a.B) return;
    __syncthreads();  // the joined results are read: the rings are free
  } while (true);
}

// A workgroup per (sequence, query head): a sequence that several pieces share is joined, its waves taking 64 / JW
// parts at a time in turn, then in the waves' order; one of no keys gets zeros; the others are finished. (One wave
// for all parts, eight at a time: one sequence of 46000 keys x 12/4 heads 33.8 / 27.7 us in all, of 12000 x 40/8
// 21.4 / 18.2; sixteen of 3000 43.3 / 43.9.)
constexpr int JW = 4;
__global__ void __launch_bounds__(JW * 64) decode_join_kernel(const DecodeArgs a) {
  __shared__ float2 wx[JW][64];
  __shared__ float wm[JW], wl[JW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)(blockIdx.x / (uint32_t)a.Hq), h = (int)(blockIdx.x % (uint32_t)a.Hq);
  int64_t all, before;
  count_tiles_of(a, lane, b, all, before);
  const int tiles = __builtin_amdgcn_readfirstlane(tiles_of(a, b));
  float x = 0.0f, y = 0.0f, L = 0.0f, M = -INFINITY;
  if (tiles > 0) {
    // tile t is in piece j when floor(all j / pieces) <= t < floor(all (j + 1) / pieces)
    const int64_t pieces = all < a.pieces ? all : a.pieces;
    const int j0 = (int)(((before + 1) * pieces - 1) / all);
    const int j1 = (int)(((before + tiles) * pieces - 1) / all);
    if (j0 == j1) return;
    const int64_t rows = (int64_t)a.pieces + a.B, row = h * rows + j0 + b;
    const float* st = a.part + a.Hq * rows * D;
    constexpr int N = 64 / JW;
    for (int i0 = N * wave; i0 <= j1 - j0; i0 += 64) {  // N parts at a time, their weights one per lane
      const int n = min(N, j1 - j0 + 1 - i0);
      const float* p = a.part + (row + i0) * D + 2 * lane;
      float2 v[N];
#pragma unroll
      for (int u = 0; u < N; ++u)
        v[u] = u < n ? *reinterpret_cast<const float2*>(p + (int64_t)u * D) : float2{0.0f, 0.0f};
      float m = -INFINITY, l = 0.0f;
      if (lane < n) {
        m = st[row + i0 + lane];
        l = st[a.Hq * rows + row + i0 + lane];
      }
      float mx = m;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      const float mn = fmaxf(M, mx);
      const float f0 = M == -INFINITY ? 0.0f : fast_exp2((M - mn) * a.scale_log2);
      const float w = m == -INFINITY ? 0.0f : fast_exp2((m - mn) * a.scale_log2);
      x *= f0;
      y *= f0;
      L = L * f0 + wave_reduce_sum(w * l);
      M = mn;
#pragma unroll
      for (int u = 0; u < N; ++u) {  // (lanes past n have weight 0)
        const float f = __shfl(w, u);
        x += f * v[u].x;
        y += f * v[u].y;
      }
    }
  }
  wx[wave][lane] = float2{x, y};
  if (lane == 0) {
    wm[wave] = M;
    wl[wave] = L;
  }
  __syncthreads();
  if (wave != 0) return;
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < JW; ++w) M = fmaxf(M, wm[w]);
  x = y = L = 0.0f;
#pragma unroll
  for (int w = 0; w < JW; ++w) {
    const float f = wm[w] == -INFINITY ? 0.0f : fast_exp2((wm[w] - M) * a.scale_log2);
    L += f * wl[w];
    x += f * wx[w][lane].x;
    y += f * wx[w][lane].y;
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  *reinterpret_cast<uint32_t*>(a.out.p + b * a.out.sl + h * a.out.sh + 2 * lane) =
      pack_bf16x2(x * inv, y * inv);
}

}  // namespace

// Pieces per key/value head (and block of 32 of its query heads): none while whole sequences give work
// enough or caches are short, else as many as run at once, two workgroups a CU, of 6 tiles or more (of 4 / 6 / 8:
// one sequence of 5000 keys x 40/8 heads 14.4 / 12.9 / 13.3 us, two of 5000 x 12/4 14.3 / 12.9 / 14.7).
// Short, whole / cut, x 40/8 heads: one sequence of 500 keys 7.4 / 9.7 us, of 1000 9.9 / 9.8, of 1500 12.2 / 10.0;
// four of 500 7.6 / 10.5, of 1000 10.6 / 11.2, of 1500 13.1 / 11.5; sixteen of 1000 15.7 / 18.9, of 1500 20.4 / 23.3.
// The rule sees the capacity, as lengths are on the device: few keys in a long cache are cut (500 in 4096 rows: the
// 9.7 us above), and from batch x units = 2 x CUs on one long sequence among short ones is not.
int decode_pieces(int64_t B, int Hq, int Hk, int64_t S, int num_splits, int cus) {
  const int64_t units = (int64_t)Hk * ((Hq / Hk + HEADS - 1) / HEADS);
  if (num_splits == 1) return 0;
  if (num_splits > 1) return (int)std::min<int64_t>(num_splits * B, 1 << 20);
  if (S <= 1024 || B * units >= 2 * cus) return 0;
  const int64_t most = std::max<int64_t>(1, 2 * cus / units), tiles = B * ((S + DT - 1) / DT);
  return (int)std::max<int64_t>(1, std::min(most, tiles / 6));
}

template <int DW>
static hipError_t run(const DecodeArgs& a, hipStream_t stream) {
  constexpr int bytes = DW * RING_B + 2 * DW * HEADS * 4;
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)decode_kernel<DW>, bytes, allowed);
  if (attr != hipSuccess) return attr;
  const int group = a.Hq / a.Hk, blocks = (group + HEADS - 1) / HEADS;
  const int64_t n = (int64_t)(a.pieces > 0 ? a.pieces : a.B) * blocks * a.Hk;
  hipLaunchKernelGGL(decode_kernel<DW>, dim3((uint32_t)n), dim3(DW * 64), bytes, stream, a);
  return hipGetLastError();
}

hipError_t launch_decode(const DecodeArgs& a, hipStream_t stream) {
  const int group = a.Hq / a.Hk, blocks = (group + HEADS - 1) / HEADS;
  // whole sequences that leave every CU one workgroup at most: eight waves in it (one sequence of 500 keys
  // x 40/8 heads 8.0 / 7.4 us with four / eight, of 1000 12.1 / 9.8; 64 of 500, two workgroups a CU, 28 / 31)
  if (a.pieces == 0 && (int64_t)a.B * blocks * a.Hk <= num_cus()) return run<8>(a, stream);
  const hipError_t e = run<4>(a, stream);
  if (e != hipSuccess || a.pieces == 0) return e;
  hipLaunchKernelGGL(decode_join_kernel, dim3((uint32_t)(a.B * a.Hq)), dim3(JW * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
