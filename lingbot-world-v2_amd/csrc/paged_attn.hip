// Attention of one query token per sequence over a paged cache (gfx950).
//
//   out[b, h] = softmax(scale q[b, h] K^T) V over the keys of a common prefix (if any), then the sequence's own:
//   all keys 0 .. len[b] - 1, or those of the selected pages; key/value head h / (Hq / Hk); no keys give 0.
//
// Bound by reading K and V once. The work of a workgroup is as in the single-token attention over whole caches: one
// key/value head, up to 32 query rows as the columns of S^T = K Q^T, 4 or 8 waves that take 32-key tiles in turn,
// each through 16 KB of LDS of its own, and join their results at the end. Here a tile is two halves of 16
// tokens, each inside one page (pages are 16 tokens or more). The pages of a wave's next 32 tiles are looked
// up at once, one half a lane, and handed to the scalar side a tile ahead.
//
// The prefix's keys are the same for the whole batch: its query rows are those of all sequences, 32 at a time, or 128
// where there are more (four waves over shared tiles of 64 keys), in one launch with the sequences' own keys. A short prefix
// is walked by every sequence before its own keys.
//
// Measured, x 40/8 heads: eight sequences of up to 46800 keys 166 us, K and V at 6.4 TB/s (a plain kernel that only reads
// reaches 5.7); 64 of up to 3600 behind a prefix of 46800 160 us, 16 of 200 (12/4 heads) behind 46800 37; one
// sequence of 500 keys 9.1 us, 3 us of it the launch and 1.5 a tile of each wave.
//
// The softmax weights are rounded to bf16 for the product with V, as the matrix instruction takes them (their sum is not):
// over many keys of like weight that is an error of the size of the result's own rounding. Distance from the 64-bit result,
// relative to its norm, where rounding that result once gives 0.0016 to 0.0017: 0.0018 for 16 branches, 0.0020 for eight
// sequences of up to 46800 keys, 0.0023 for 64 branches off 46800.
//
// A half's rows past its last key copy that key (or the other half's), so the products never meet what lies
// behind a sequence; V's of them are zeros before the product, as their weight of 0 would make NaN of a copy of an infinite
// value. A page outside the cache makes its keys' scores NaN. Scores that are all -infinity give NaN (0 / 0), no keys 0.

#include <algorithm>

#include "capi_util.h"
#include "packed_loop.h"
#include "paged.h"
#include "sequence_tiles.h"

namespace lbw {
namespace {

constexpr int DT = 32;                      // keys per tile
constexpr int HT = DT / 2;                  // keys per half
static_assert(HT == HALF_KEYS, "half_at looks up half a tile");
constexpr int DT_B = DT * PK_ROWB;          // 8 KB
constexpr int RING_B = 2 * DT_B;            // per wave: K, V
constexpr int NCOPY = DT_B / 1024;          // copies per lane for K or V of a tile
constexpr int HEADS = 32;                   // query rows per workgroup (as own_units counts them)
enum Kind { DENSE, SPARSE, PREFIX };
constexpr int P_LIST = 4096;                // table entries of a piece of the prefix (tile form)
constexpr int PREFIX_LDS = FWD_LDS + 4 * P_LIST;
typedef __attribute__((address_space(3))) int32_t lds_i32;

// A sequence's keys: its length, limited to what its row of the table holds.
__device__ __forceinline__ int keys_of(const PagedAttnArgs& a, int b) {
  const int64_t cap = (int64_t)a.pt.width << a.pt.shift;
  const int n = a.lens[b];
  return n < 0 ? 0 : (n > cap ? (int)cap : n);
}
__device__ __forceinline__ int tiles_of(const PagedAttnArgs& a, int b) { return (int)(((int64_t)keys_of(a, b) + DT - 1) / DT); }
__device__ __forceinline__ int64_t prefix_keys(const PagedAttnArgs& a) {
  int64_t n = a.p_len != nullptr ? a.p_len[0] : a.p_max;
  return n < 0 ? 0 : (n > a.p_max ? a.p_max : n);
}
// 1 / L of a row with reference M: 0 without keys (M = -inf), NaN where they give no sum (scores of -infinity alone).
__device__ __forceinline__ float inverse_sum(float M, float L) {
  return L > 0.0f ? 1.0f / L : (M == -INFINITY ? 0.0f : __uint_as_float(0x7fc00000u));
}
// Entries of a list of selected pages: those before the first negative one.
__device__ __forceinline__ int list_length(const int32_t* sel, int n, int lane) {
  constexpr int U = 4;  // (loads under way at once)
  for (int i0 = 0; i0 < n; i0 += 64 * U) {
    int32_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = i0 + 64 * u + lane < n ? sel[i0 + 64 * u + lane] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t stop = __ballot(x[u] < 0);
      if (stop != 0) return i0 + 64 * u + __ffsll((unsigned long long)stop) - 1;
    }
  }
  return n;
}

// Workgroup `id` of those for one kind of keys: key/value head (fastest), block of query rows, piece.
template <int DW, Kind KIND>  // waves per workgroup
__device__ __forceinline__ void attend_pages(const PagedAttnArgs& a, uint32_t id, unsigned char* lds) {
  constexpr int DEC_LDS = DW * RING_B;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int group = a.group;
  const int64_t rows_all = KIND == PREFIX ? (int64_t)a.B * group : group;  // query rows of a key/value head
  const uint32_t blocks = (uint32_t)((rows_all + HEADS - 1) / HEADS);
  const int kv = id % (uint32_t)a.Hk;
  id /= (uint32_t)a.Hk;
  const int64_t r0 = (int64_t)(id % blocks) * HEADS;
  const int piece = id / blocks;
  const int nr = (int)(rows_all - r0 < HEADS ? rows_all - r0 : HEADS);
  const bool end_to_end = KIND == DENSE && DW == 4 && a.pieces > 0;  // (eight waves: whole sequences)
  const int splits = KIND == PREFIX ? a.p_splits : a.splits;

  // this workgroup's tiles [at, end) of the batch laid end to end, from sequence b on
  int b = KIND == PREFIX ? 0 : piece / (end_to_end ? 1 : splits);
  const int split = end_to_end ? 0 : (KIND == PREFIX ? piece : piece % splits);
  int64_t at = 0, end = 1, before = 0;
  if (end_to_end) {
    int64_t all, none;
    count_tiles_of(a.B, [&](int s) { return tiles_of(a, s); }, lane, 0, all, none);
    // (no more pieces than tiles: an empty one between two parts of a sequence would leave a row unwritten)
    const int64_t pieces = all < a.pieces ? all : a.pieces;
    if (piece >= pieces) return;
    at = all * piece / pieces;
    end = all * (piece + 1) / pieces;
    b = find_sequence(a.B, [&](int s) { return tiles_of(a, s); }, lane, at, before);
    if (b >= a.B) return;
  }

  const int ring = (int)lds_addr(lds) + RING_B * wave;
  const int ka = row_address(ring, l32, hl), va = tr_address(ring + DT_B, lane, hl);
  // copy i of a tile: rows 4 i + lane / 16, chunk (lane % 16) ^ swz(row); rows i and i + 4 share the chunk
  const int crow = lane >> 4, ccol = ((lane & 15) ^ swz(lane >> 4)) * 16;
  const uint32_t koff = (uint32_t)crow * (uint32_t)(a.k.sl * 2), voff = (uint32_t)crow * (uint32_t)(a.v.sl * 2);
  const float c = sreg(a.scale_log2);
  const int shift = a.pt.shift, mask = (1 << shift) - 1;
  const int64_t own = own_rows(a), rows = all_rows(a);

  do {
    // query row x of the workgroup: its sequence and head
    auto seq_of = [&](int x) { return KIND == PREFIX ? (int)((r0 + x) / group) : b; };
    auto head_of = [&](int x) { return kv * group + (int)(KIND == PREFIX ? (r0 + x) % group : r0 + x); };
    u32x4 qf[8];
    {
      const int x = l32 < nr ? l32 : nr - 1;
      const uint16_t* p = a.q.p + seq_of(x) * a.q.sl + head_of(x) * a.q.sh + 8 * hl;
#pragma unroll
      for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const u32x4*>(p + 16 * s);
    }
    // the list of this sequence's pages: `count` entries of 2^shift tokens, `len` keys in all
    const int64_t len = KIND == PREFIX ? scalar64(prefix_keys(a)) : __builtin_amdgcn_readfirstlane(keys_of(a, b));
    const int32_t* const table = KIND == PREFIX ? a.p_table : a.pt.p + b * a.pt.sb;
    const int32_t* const sel = KIND == SPARSE ? a.sel + ((int64_t)b * a.Hk + kv) * a.n_sel : nullptr;
    const int64_t own_span =
        KIND == SPARSE
            ? (len > 0 ? (int64_t)__builtin_amdgcn_readfirstlane(list_length(sel, a.n_sel, lane)) << shift : 0)
            : len;
    // a short prefix's keys, in halves of their own, come before the sequence's
    const int64_t p_keys = KIND != PREFIX && a.p_inline != 0 ? scalar64(prefix_keys(a)) : 0;
    const int64_t pre = (p_keys + HT - 1) / HT * HT, span = pre + own_span;
    const int tiles = (int)((span + DT - 1) / DT);
    // this sequence's tiles of the piece
    int s0 = 0, s1 = tiles;
    if (end_to_end) {
      s0 = (int)(at - before);
      s1 = (int)(end - before < tiles ? end - before : tiles);
    } else if (splits > 1) {
      s0 = (int)((int64_t)tiles * split / splits);
      s1 = (int)((int64_t)tiles * (split + 1) / splits);
    }

    // halves of tiles base, base + DW, ..: tile i's first half in lane i, its second in lane 32 + i
    auto look_up = [&](int base) {
      const int64_t pos = ((int64_t)base + (int64_t)l32 * DW) * DT + HT * hl;
      if (pos < pre) return half_at(nullptr, p_keys, a.p_table, a.p_width, shift, a.pt.pages, p_keys, pos);
      return half_at(sel, own_span, table, KIND == PREFIX ? a.p_width : a.pt.width, shift, a.pt.pages, len, pos - pre);
    };
    Half list = {0, 0}, h0, h1;  // h0, h1: the halves of the tile that is fetched next, scalar
    int listed = 0;              // tiles of the list that are used up
    auto next_halves = [&](int t) {
      if ((listed & 31) == 0) {
        list = look_up(t);
        // (waited for here, once in 32 tiles: a load that may be pending after the branch would be waited for, and
        // the copies with it, at every tile)
        asm volatile("" : "+v"(list.page), "+v"(list.keys));
      }
      const int i = listed & 31;
      h0.page = __builtin_amdgcn_readlane(list.page, i);
      h0.keys = __builtin_amdgcn_readlane(list.keys, i);
      h1.page = __builtin_amdgcn_readlane(list.page, i + 32);
      h1.keys = __builtin_amdgcn_readlane(list.keys, i + 32);
      ++listed;
    };
    auto issue = [&](const PageRows& src, uint32_t off, int t, uint32_t to) {
      const unsigned char* base = reinterpret_cast<const unsigned char*>(src.p + kv * src.sh);
      const int64_t sl = src.sl * 2, sp = src.sp * 2;
      // (places behind a prefix count from its end)
      const int64_t at0 = (int64_t)t * DT, at1 = at0 + HT;
      const int in = (int)((at0 < pre ? at0 : at0 - pre) & mask), in1 = (int)((at1 < pre ? at1 : at1 - pre) & mask);
      const int n0 = h0.keys & (BAD_PAGE - 1), n1 = h1.keys & (BAD_PAGE - 1);
      const unsigned char* p0 = base + h0.page * sp + in * sl;
      const unsigned char* p1 = base + h1.page * sp + in1 * sl;
      // a half without keys copies the other's last one (a tile without any: anything, it is not used)
      // (scalar: the compiler does not see that an address is the same in every lane)
      auto scalar = [](const unsigned char* p) { return (const unsigned char*)(uintptr_t)scalar64((int64_t)(uintptr_t)p); };
      const unsigned char* b0 = scalar(n0 > 0 || n1 == 0 ? p0 : p1);
      const unsigned char* b1 = scalar(n1 > 0 || n0 == 0 ? p1 : p0);
      const uint32_t last0 = (uint32_t)((n0 > 0 ? n0 : (n1 > 0 ? n1 : 1)) - 1) * (uint32_t)sl;
      const uint32_t last1 = (uint32_t)((n1 > 0 ? n1 : (n0 > 0 ? n0 : 1)) - 1) * (uint32_t)sl;
#pragma unroll
      for (int i = 0; i < NCOPY; ++i) {  // (rows past the last key copy it)
        const uint32_t row = min(off + 4 * (i & 3) * (uint32_t)sl, i < 4 ? last0 : last1);
        // (own keys past the caches: eight of up to 46800 x 40/8 heads 186 to 165 us, 12/12 of 14040 95 to 84, selected pages too;
        // the prefix's, which other rows' workgroups read, not: 16 of 3000 off 46800 67 to 97)
        if constexpr (KIND == PREFIX) dma16_guarded(i < 4 ? b0 : b1, row + (ccol ^ ((i & 3) << 4)), to + 1024 * i);
        else dma16_past(i < 4 ? b0 : b1, row + (ccol ^ ((i & 3) << 4)), to + 1024 * i);
      }
    };
    auto issue_k = [&](int t) { issue(a.k, koff, t, (uint32_t)ring); };
    auto issue_v = [&](int t) { issue(a.v, voff, t, (uint32_t)ring + DT_B); };
    static_assert(NCOPY == 8, "the counts below are a tile's copies");

    floatx16 o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db) zero(o[db]);
    float m = M_INIT, l = 0.0f;
    __builtin_amdgcn_s_waitcnt(0x0070);  // the query is there: only tile copies are counted below
    int t = s0 + wave, k0 = 0, k1 = 0;   // keys of the current tile's halves
    int any = 0;                         // whether the wave had keys
    if (t < s1) {
      next_halves(t);
      issue_k(t);
      issue_v(t);
    }
#pragma unroll 1
    for (; t < s1; t += DW) {
      const bool more = t + DW < s1;
      k0 = h0.keys;
      k1 = h1.keys;
      any |= k0 | k1;
      if (more) next_halves(t + DW);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // K is there (V may be on its way)
      floatx16 s;
      zero(s);
#pragma unroll
      for (int d = 0; d < 8; ++d) s = mfma32x32x16(read_row(ka, d, 0), qf[d], s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its reads are over before K is overwritten
      if (more) issue_k(t + DW);
      if (k0 != HT || k1 != HT) {
        // registers 0 .. 7 are keys of the first half, 8 .. 15 of the second
        const int n0 = (k0 & (BAD_PAGE - 1)) - 4 * hl, n1 = (k1 & (BAD_PAGE - 1)) - 4 * hl;
        const float bad0 = k0 >= BAD_PAGE ? __uint_as_float(0x7fc00000u) : 0.0f;
        const float bad1 = k1 >= BAD_PAGE ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = acc_row(r & 7) < (r < 8 ? n0 : n1) ? s[r] + (r < 8 ? bad0 : bad1) : -INFINITY;
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
      if (((k0 | k1) & (2 * BAD_PAGE - 1)) != 0) {  // (a tile without keys holds anything)
        if (k0 != HT || k1 != HT) {  // (16 lanes a row, so the writes meet no bank conflict)
#pragma unroll
          for (int i = 0; i < NCOPY; ++i)
            if (4 * (i & 3) + crow >= ((i < 4 ? k0 : k1) & (BAD_PAGE - 1)))
              *(lds_u32x4*)(uintptr_t)(ring + DT_B + 1024 * i + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int mm = 0; mm < 2; ++mm) o[db] = mfma32x32x16(read_tr(va, db, mm, 0), pf[mm], o[db]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) issue_v(t + DW);
    }
    l = wave_sum_xor32(l);
    // O^T as rows [row][128] fp32 into the wave's LDS, m and l behind the rings
    float* const sm = reinterpret_cast<float*>(lds + DEC_LDS);
    float* const sl = sm + DW * HEADS;
    if (hl == 0) {  // (no keys: a reference of -inf, weight 0; scores of -inf alone: the first reference, a sum of 0)
      sm[wave * HEADS + l32] = any != 0 ? m : -INFINITY;
      sl[wave * HEADS + l32] = l;
    }
    float* mine = reinterpret_cast<float*>(lds + RING_B * wave);
    if (l32 < nr) {
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
    const bool whole = KIND != PREFIX && s1 - s0 == tiles && a.p_splits == 0 && (end_to_end || splits == 1);
    for (int x = threadIdx.x; x < nr * (D / 4); x += DW * 64) {  // 4 values of one row at a time
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
      const int sq = seq_of(hh), head = head_of(hh);
      if (whole) {
        const float inv = inverse_sum(M, L);
        u32x2 w;
        w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
        w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<u32x2*>(a.out.p + sq * a.out.sl + head * a.out.sh + dq) = w;
      } else {
        // (end to end: piece + b, the parts of a head in the order of their keys, each in a row of its own, as the
        // next part has another piece or a later sequence, or both)
        const int64_t part = KIND == PREFIX ? own + (int64_t)sq * splits + split
                                            : (end_to_end ? (int64_t)piece + b : (int64_t)b * splits + split);
        const int64_t row = head * rows + part;
        *reinterpret_cast<floatx4*>(a.part + row * D + dq) = acc;
        if (dq == 0) {
          float* st = a.part + a.Hq * rows * D;
          st[row] = M;
          st[a.Hq * rows + row] = L;
        }
      }
    }
    if (!end_to_end) return;
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

// A piece of the prefix for 128 query rows of a key/value head: the packed attention's walk, 4 waves of 32 rows over
// shared tiles of 64 keys, each wave copying the 16 tokens of a tile that lie in one page. A page outside the cache
// becomes keys of NaN. `id`: piece, block of rows, head, the head fastest, so that a piece's blocks of rows run beside
// each other on one XCD.
__device__ __forceinline__ void prefix_tiles(const PagedAttnArgs& a, uint32_t id, unsigned char* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int group = a.group;
  const int64_t rows_all = (int64_t)a.B * group;
  const uint32_t blocks = (uint32_t)((rows_all + PK_BLOCK - 1) / PK_BLOCK);
  const int kv = id % (uint32_t)a.Hk;
  id /= (uint32_t)a.Hk;
  const int64_t r0 = (int64_t)(id % blocks) * PK_BLOCK + 32 * wave;  // this wave's first row
  const int piece = id / blocks;
  const int nr = (int)(rows_all - r0 < 32 ? rows_all - r0 : 32);      // and how many it has (0 or less: none)
  const int len = (int)scalar64(prefix_keys(a)), shift = a.pt.shift, mask = (1 << shift) - 1;
  const int n_tiles = (len + BN - 1) / BN;
  const int t0 = (int)((int64_t)n_tiles * piece / a.p_splits);
  const int T = (int)((int64_t)n_tiles * (piece + 1) / a.p_splits) - t0;

  u32x4 qf[8];
  {
    const int64_t row = r0 + l32 < rows_all ? r0 + l32 : rows_all - 1;  // this lane's query row
    const uint16_t* p = a.q.p + row / group * a.q.sl + (kv * group + row % group) * a.q.sh + 8 * hl;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const u32x4*>(p + 16 * s);
  }
  // the pages of the piece's table entries, behind the tiles in LDS (-1: outside the cache)
  const int e0 = (int)(((int64_t)t0 * BN) >> shift), n_pages = T > 0 ? (int)(((int64_t)(t0 + T) * BN - 1) >> shift) - e0 + 1 : 0;
  const int list = (int)lds_addr(lds) + FWD_LDS;
  for (int i = threadIdx.x; i < n_pages; i += PK_WAVES * 64)
    *(lds_i32*)(uintptr_t)(list + 4 * i) =
        page_at(a.p_table, a.p_width, shift, a.pt.pages, (int64_t)(e0 + i) << shift);
  __syncthreads();
  // a wave's share of a tile: 16 tokens of one page; one without keys copies the prefix's last one
  const int share = 16 * wave;
  const int end = len > 0 ? len - 1 : 0;
  const int crow = lane >> 4, ccol = ((lane & 15) ^ swz(lane >> 4)) * 16;
  const uint32_t koff = (uint32_t)crow * (uint32_t)(a.k.sl * 2), voff = (uint32_t)crow * (uint32_t)(a.v.sl * 2);
  const uint32_t dst = lds_addr(lds) + 1024 * PK_NDMA * wave;
  auto page_of = [&](int u) {  // (read ahead of its use)
    int pos = (t0 + u) * BN + share;
    pos = pos < len ? pos : end;
    return *(const lds_i32*)(uintptr_t)(list + 4 * ((pos >> shift) - e0));
  };
  auto issue = [&](const PageRows& src, uint32_t off, int page, int u, uint32_t to, bool is_k) {
    const int pos = (t0 + u) * BN + share;
    if (page < 0) {
      if (is_k) {
        // (opaque here and below: nothing of this is worth registers in the loop, which has none left)
        const uint32_t nan = opaque(0x7fc07fc0);
        const int at = opaque(16 * lane);
#pragma unroll
        for (int i = 0; i < PK_NDMA; ++i)
          *(lds_u32x4*)(uintptr_t)(to + 1024 * i + at) = u32x4{nan, nan, nan, nan};
        return;
      }
      page = 0;
    }
    const int64_t sl = src.sl * 2;
    const int in = (pos < len ? pos : end) & mask, more = len - 1 - pos;  // tokens behind the share's first one
    const unsigned char* b = reinterpret_cast<const unsigned char*>(src.p + kv * src.sh) + page * (src.sp * 2) + in * sl;
    const uint32_t last = (uint32_t)(more < HT - 1 ? (more > 0 ? more : 0) : HT - 1) * (uint32_t)sl;
    const int col = opaque(ccol);
    if (!is_k && more < HT - 1) {  // (the last tile: zeros behind the last key)
      const int at = opaque(16 * lane);
#pragma unroll
      for (int i = 0; i < PK_NDMA; ++i) {
        const int row = (at >> 8) + 4 * i;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (row <= more) x = *reinterpret_cast<const u32x4*>(b + row * sl + (col ^ (i << 4)));
        *(lds_u32x4*)(uintptr_t)(to + 1024 * i + at) = x;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < PK_NDMA; ++i)
      dma16_guarded(b, min(off + 4 * i * (uint32_t)sl, last) + (col ^ (i << 4)), to + 1024 * i);
  };
  // K of tile u + 1 goes ahead of V of tile u: the page of the share before is kept
  int ahead = T > 0 ? page_of(0) : 0, now = 0, prev = 0;
  auto issue_k = [&](int u) {
    prev = now;
    now = __builtin_amdgcn_readfirstlane(ahead);
    issue(a.k, koff, now, u, dst + (u & 1) * PK_TILE_B, true);
    if (u + 1 < T) ahead = page_of(u + 1);
  };
  auto issue_v = [&](int u) {
    issue(a.v, voff, u > 0 && u + 1 < T ? prev : now, u, dst + V_AT + (u & 1) * PK_TILE_B, false);
  };
  floatx16 o[4];
  float m, l;
  if (nr <= 0) {
    copy_tiles(lds, wave, lane, T, issue_k, issue_v);
    return;
  }
  // (every wave that gets here needs all tiles: a count of its own would cost 60 registers)
  attend_tiles(lds, wave, lane, qf, sreg(a.scale_log2), t0, T, T, len, len, issue_k, issue_v, o, m, l);
  l = wave_sum_xor32(l);
  if (l32 >= nr) return;
  // (the lane hidden: the row's place is worked out anew, not kept in registers all the way)
  const int64_t row = r0 + opaque(l32), rows = all_rows(a);
  const int64_t part = (kv * group + row % group) * rows + own_rows(a) + row / group * a.p_splits + piece;
  float* const dst_o = a.part + part * D + 4 * hl;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4*>(dst_o + 32 * db + 8 * g) =
          floatx4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
  if (hl == 0) {
    float* st = a.part + a.Hq * rows * D;
    st[part] = T > 0 ? m : -INFINITY;
    st[a.Hq * rows + part] = l;
  }
}

template <int DW, Kind KIND>
__global__ void __launch_bounds__(DW * 64, 2) paged_kernel(const PagedAttnArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  attend_pages<DW, KIND>(a, blockIdx.x, lds);
}

// The prefix (TILES: 128 query rows at a time) and the sequences' own keys in one launch: their workgroups take turns,
// in proportion, so that a CU has some of each. The prefix's matrix products then run while own keys are read.
template <bool TILES, Kind KIND>
__global__ void __launch_bounds__(4 * 64, 2) paged_both_kernel(const PagedAttnArgs a, uint32_t p_units, uint32_t units) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const uint32_t unit = blockIdx.x / (uint32_t)a.Hk, kv = blockIdx.x % (uint32_t)a.Hk;
  const uint32_t before = (uint32_t)((uint64_t)unit * p_units / units);  // units of the prefix among those before
  if ((uint32_t)((uint64_t)(unit + 1) * p_units / units) > before) {
    if constexpr (TILES) prefix_tiles(a, before * a.Hk + kv, lds);
    else attend_pages<4, PREFIX>(a, before * a.Hk + kv, lds);
  } else {
    attend_pages<4, KIND>(a, (unit - before) * a.Hk + kv, lds);
  }
}

// A workgroup per (sequence, query head): the parts of its own keys, then the prefix's, joined, its waves taking
// 64 / JW parts at a time in turn, then in the waves' order. No parts: zeros (or, end to end without a prefix, a
// result that one piece has written already).
constexpr int JW = 4;
__global__ void __launch_bounds__(JW * 64) paged_join_kernel(const PagedAttnArgs a) {
  __shared__ float2 wx[JW][64];
  __shared__ float wm[JW], wl[JW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)(blockIdx.x / (uint32_t)a.Hq), h = (int)(blockIdx.x % (uint32_t)a.Hq);
  const int64_t own = own_rows(a), rows = all_rows(a);
  int64_t first = (int64_t)b * a.splits;  // own parts [first, first + n_own)
  int n_own = a.splits;
  if (a.pieces > 0) {
    int64_t all, before;
    count_tiles_of(a.B, [&](int s) { return tiles_of(a, s); }, lane, b, all, before);
    const int tiles = __builtin_amdgcn_readfirstlane(tiles_of(a, b));
    n_own = 0;
    if (tiles > 0) {
      // tile t is in piece j when floor(all j / pieces) <= t < floor(all (j + 1) / pieces)
      const int64_t pieces = all < a.pieces ? all : a.pieces;
      const int j0 = (int)(((before + 1) * pieces - 1) / all);
      const int j1 = (int)(((before + tiles) * pieces - 1) / all);
      if (j0 == j1 && a.p_splits == 0) return;
      first = j0 + b;
      n_own = j1 - j0 + 1;
    }
  }
  const int n_all = n_own + a.p_splits;
  // part i's row
  auto row_of = [&](int i) {
    return h * rows + (i < n_own ? first + i : own + (int64_t)b * a.p_splits + (i - n_own));
  };
  const float* st = a.part + a.Hq * rows * D;
  float x = 0.0f, y = 0.0f, L = 0.0f, M = -INFINITY;
  constexpr int N = 8;
  for (int i0 = N * wave; i0 < n_all; i0 += N * JW) {  // N parts at a time, their weights one per lane
    const int n = min(N, n_all - i0);
    float2 v[N];
#pragma unroll
    for (int u = 0; u < N; ++u)
      v[u] = u < n ? *reinterpret_cast<const float2*>(a.part + row_of(i0 + u) * D + 2 * lane) : float2{0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    if (lane < n) {
      m = st[row_of(i0 + lane)];
      l = st[a.Hq * rows + row_of(i0 + lane)];
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
  const float inv = inverse_sum(M, L);
  *reinterpret_cast<uint32_t*>(a.out.p + b * a.out.sl + h * a.out.sh + 2 * lane) =
      pack_bf16x2(x * inv, y * inv);
}

constexpr int lds_bytes(int waves) { return waves * RING_B + 2 * waves * HEADS * 4; }

template <int DW, Kind KIND>
hipError_t run(const PagedAttnArgs& a, int64_t units, hipStream_t stream) {
  constexpr int bytes = lds_bytes(DW);
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)paged_kernel<DW, KIND>, bytes, allowed);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((paged_kernel<DW, KIND>), dim3((uint32_t)(units * a.Hk)), dim3(DW * 64), bytes, stream, a);
  return hipGetLastError();
}

template <bool TILES, Kind KIND>
hipError_t run_both(const PagedAttnArgs& a, int64_t units, hipStream_t stream) {
  constexpr int bytes = TILES ? std::max(PREFIX_LDS, lds_bytes(4)) : lds_bytes(4);
  static LdsAllowed allowed;
  const hipError_t attr = allow_lds((const void*)paged_both_kernel<TILES, KIND>, bytes, allowed);
  if (attr != hipSuccess) return attr;
  const int64_t p_units = prefix_units(a);
  hipLaunchKernelGGL((paged_both_kernel<TILES, KIND>), dim3((uint32_t)((p_units + units) * a.Hk)), dim3(4 * 64), bytes,
                     stream, a, (uint32_t)p_units, (uint32_t)(p_units + units));
  return hipGetLastError();
}

}  // namespace

// How the keys are cut. Own ones: whole sequences where they keep the chip busy or are short, else the batch's keys in
// equal pieces, a workgroup a CU (two: 0 to 5 % slower); the longer for that the more sequences x key/value heads there
// are, up to one a CU, and shorter again up to half as many more, which would leave most of the CUs idle while they end.
// Whole / in pieces, x 40/8 heads, lengths from a third of the longest up to it, from memory: one sequence of 1100 keys
// 11.6 / 14.4 us, of 1300 16.2 / 13.9; four of 1000 14.7 / 16.0, of 1300 17.0 / 15.9; eight of 1000 14.7 / 16.3, of 1500
// 19.4 / 18.4; 16 of 1600 20.6 / 21.6, of 2000 25.2 / 23.5, of 4000 45.7 / 38.9; 20 of 2400 30.4 / 31.7, of 3200 38.0 /
// 35.9; 24 of 3200 40.2 / 41.3, of 4000 49.6 / 48.6; 32 of 4000 60.6 / 63.6, of 5000 74.7 / 73.9; 33 of 1200 28.7 / 30.4,
// of 1700 41.7 / 36.6, of 3200 65.6 / 57.0; 36 of 1200 31.8 / 32.2, of 1700 42.7 / 38.9, of 3200 70.0 / 61.3; 40 of 1200
// 32.5 / 33.6, of 1700 44.8 / 42.1, of 3200 77.8 / 67.7; 48 of 1700 47.2 / 49.3, of 2400 61.6 / 61.4, of 3200 83.7 / 79.1;
// 50 of 2400 62.5 / 62.6, of 3200 84.6 / 81.6; 56 of 2400 67.6 / 70.7, of 3500 98.6 / 96.7; 64 of 2400 72.5 / 76.6, of 4000
// 115 / 116, of 8000 221 / 211; 128 of 2400 135 / 140, of 4000 218 / 214.
// Selected pages: equal lengths, so pieces pay sooner, of 4 tiles or more (and a whole list each where there are more
// lists than half the CUs). Whole / in pieces, x 40/8 heads: 512 keys for one sequence 9.3 / 11.0 us, for 8 11.0 / 11.1, for 16
// 11.6 / 12.5; 768 12.3 / 11.2, 13.4 / 12.7, 14.0 / 14.5; 1024 14.7 / 11.3, 15.8 / 13.4, 16.7 / 16.6; 2560 28.0 / 10.9, 30.8 / 20.6,
// 33.1 / 29.3; a workgroup a CU / two: 5760 for 8 35.4 / 35.5, 6400 for 4 23.1 / 23.7, for 24 88.5 / 100.6.
// With a prefix (measured before own keys went past the caches, which changes both sides alike; shares by 0.5, 0.6,
// 0.7 and 0.8 of own keys then gave 167, 166, 160 and 177 us for 64 of 3600 off 46800), places shared out by tiles:
// 4 of up to 1600 off 14040 keys x 40/8 heads, 20 pieces of the prefix and 12 of own keys 22.2 us, 32 and 32 25.8; 8
// of 3600 off 6000 x 12/4, 9 and 55 21.2, 64 and 64 28.2; 64 of 3600 off 46800 x 40/8 (128 rows at a time), 10 and
// 34 163, 21 and 64 185, 5 and 17 205; 26 of 1500 off 14040 x 40/8 16 and 32 40.4, 8 and 16 45.8; 30 of 1500 off
// 10000 x 16/2, 32 and 64 23.5, 64 and 128 27.6. Whole sequences: 16 of 200 off 6000 x 12/4, 24 pieces (one
// workgroup a CU) 14.4, 48 16.6; off 46800 20 35.9, 48 39.6; 16 of 200 off 14040 x 40/8 (128 sequences x heads), 4
// pieces 47.1, 16 (two a CU) 26.6. Ten of 472 off 4254 x 40/40 (400), 2 pieces 49.1, 6 36.5; 60 of 300 off 10000 x
// 12/12 (720), one 122.7, 21 44.8; 128 rows at a time: 29 of 102 off 9496 x 40/8 (232), 17 pieces 30.5, 24 38.6; 64
// of 200 off 14040 (512), 10 58.3, 16 53.6. Pieces of 4 tiles or more, of 6: 4 of 40 off 1560 x 12/4 12.3 / 13.3,
// one of 3000 x 40/8 11.7 / 13.0; of 128 rows, of 4 or 8: 41 of 800 off 3366 x 12/4 25.3 / 20.3, 64 of 500 off 6000
// 30.8 / 25.9.
// 32 / 128 query rows at a time: 8 of 1500 off 14040 x 40/8 (40 rows) 30.9 / 35.6, 20 (100) 42.5 / 46.5, 40 (200) 65.6 /
// 54.4; 46800, 1000 own x 12/4, 24 rows 34.5 / 36.6, 60 rows 44.0 / 43.0, 78 rows 49.3 / 51.8, 99 rows 58.5 / 54.8.
void plan_paged(PagedAttnArgs* a, int num_splits, int cus) {
  const int64_t group = a->Hq / a->Hk, units = a->Hk * ((group + HEADS - 1) / HEADS), seqs = a->B * units;
  a->splits = 1;
  a->pieces = a->p_splits = 0;
  if (a->B == 0) return;
  // pieces of `tiles` tiles for `places` workgroups, `each` of them a piece, of `least` tiles or more
  auto cut = [&](int64_t tiles, int64_t places, int64_t each, int64_t least) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(places / each, tiles / least));
  };
  const int64_t cap = (int64_t)a->pt.width << a->pt.shift;
  const int64_t keys = a->sel != nullptr ? (int64_t)a->n_sel << a->pt.shift : cap;
  const int64_t own_tiles = (keys + DT - 1) / DT;  // of a sequence
  // (with a prefix, whose results are joined anyway, pieces cost less)
  const int64_t limit = a->p_max > 0                                ? 1024
                        : a->sel != nullptr                         ? 512 + 3 * seqs
                        : seqs <= cus                               ? 1150 + 3200 * seqs * seqs / ((int64_t)cus * cus)
                        : 2 * seqs <= 3 * cus                       ? 1500
                                                                    : 3500;
  const bool whole = num_splits == 1 || (num_splits == 0 && keys <= limit);
  int64_t own_places = cus;
  // A short prefix: every sequence walks it itself, one launch without a join. Apart / so: 16 sequences x 40/8 heads, 400 keys
  // and 20 own 14.8 / 9.9 us, 500 and 500 16.1 / 13.6, 1200 and 40 18.5 / 14.4; 4 x 12/12 14.2 / 9.8, 15.0 / 14.3, 13.9 / 15.0; more
  // than one a CU, 32 x 12/12 14.7 / 13.7, 21.5 / 23.7, 18.0 / 24.0, 64 x 12/12 21.5 / 21.4, 32.2 / 41.6, 24.5 / 39.3.
  a->p_inline = a->p_max > 0 && num_splits == 0 && a->p_max + keys <= (seqs <= cus ? 1100 : 450);
  if (a->p_inline) return;
  if (a->p_max > 0) {
    const int64_t rows = a->B * group, p_tiles = (a->p_max + DT - 1) / DT;
    a->p_block = rows > 3 * HEADS ? PK_BLOCK : HEADS;
    const int64_t each = a->Hk * ((rows + a->p_block - 1) / a->p_block);
    const bool wide = a->p_block == PK_BLOCK;
    // tiles of all workgroups; own ones are counted to the longest sequence's end, 0.7 of that beside 128 rows at a
    // time, whose few pieces are the last to end (64 of 3600 off 46800, 40/8 heads: 163 us, 7 pieces at 1.0 215)
    const int64_t of_prefix = p_tiles * each, of_own = own_tiles * seqs * (wide ? 7 : 10) / 10;
    int64_t places;
    if (whole) {
      // a workgroup a CU, whole sequences included; two where those would leave the prefix less than 0.7 of the CUs; one a
      // CU (or three for two) for the prefix alone where they fill the chip by themselves
      const int64_t one = std::max<int64_t>(0, cus - seqs) / each * each;
      places = !wide && 10 * one >= 7 * cus ? one : std::max<int64_t>(2 * cus - seqs, wide && seqs > cus ? 3 * cus / 2 : cus);
    } else {
      // a workgroup a CU, shared out by their tiles; two where each still gets 16 tiles (of 128 rows, which alone on
      // a CU wait most of the time) or 32
      const int64_t all = of_prefix + of_own >= (wide ? 32 : 64) * cus ? 2 * cus : cus;
      places = all * of_prefix / (of_prefix + of_own) + (wide ? each / 2 : 0);
      own_places = all - std::max<int64_t>(1, places / each) * each;
    }
    a->p_splits = cut(p_tiles, places, each, wide ? 8 : 4);
    if (num_splits > 0) a->p_splits = num_splits;
    // (a piece's table entries fit their place: whole tiles of 64 keys, an entry more where a piece ends in a page)
    const int64_t tiles = (a->p_max + BN - 1) / BN, most = ((int64_t)(P_LIST - 1) << a->pt.shift) / BN;
    if (a->p_block == PK_BLOCK) a->p_splits = (int)std::max<int64_t>(a->p_splits, (tiles + most - 1) / most);
  }
  if (a->sel != nullptr) {
    if (num_splits > 0) a->splits = num_splits;
    else if (!whole) a->splits = cut(own_tiles, own_places, seqs, 4);
  } else if (num_splits > 1) {
    a->pieces = (int)std::min<int64_t>((int64_t)num_splits * a->B, 1 << 20);
  } else if (!whole) {
    a->pieces = cut(a->B * own_tiles, own_places, units, 4);
  }
}

hipError_t launch_paged(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t n = own_units(a);
  hipError_t e;
  if (a.p_splits > 0) {
    const bool tiles = a.p_block == PK_BLOCK;
    if (a.sel != nullptr) e = tiles ? run_both<true, SPARSE>(a, n, stream) : run_both<false, SPARSE>(a, n, stream);
    else e = tiles ? run_both<true, DENSE>(a, n, stream) : run_both<false, DENSE>(a, n, stream);
  } else {
    // whole sequences that leave every CU one workgroup at most: eight waves in it
    const bool wide = a.pieces == 0 && n * a.Hk <= num_cus();
    if (a.sel != nullptr) e = wide ? run<8, SPARSE>(a, n, stream) : run<4, SPARSE>(a, n, stream);
    else e = wide ? run<8, DENSE>(a, n, stream) : run<4, DENSE>(a, n, stream);
  }
  if (e != hipSuccess || !has_parts(a)) return e;
  hipLaunchKernelGGL(paged_join_kernel, dim3((uint32_t)((int64_t)a.B * a.Hq)), dim3(JW * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
