// What the packed attention kernels share: work items, tile staging and masks.
//
// A 64-row tile of a bf16 operand lies in LDS as 64 rows of 256 bytes, 16-byte chunk c of row r at
// chunk c ^ swz(r) (attn_tiles.h), so that both the row reads (A operand, ds_read_b128) and the
// transpose reads (ds_read_b64_tr_b16) are free of bank conflicts.
#pragma once

#include "attn_tiles.h"
#include "packed.h"

namespace lbw {

constexpr int PK_WAVES = PK_BLOCK / 32;         // waves per workgroup, 32 rows each
constexpr int PK_ROWB = D * 2;                  // bytes per row in LDS
constexpr int PK_TILE_B = BN * PK_ROWB;         // 16 KB
constexpr int PK_NDMA = PK_TILE_B / (PK_WAVES * 64 * 16);  // 16-byte copies per lane and tile

// A work item's fields, in scalar registers.
struct PackedItem {
  int row0, rows, pos0, other0, other_len, bound, shift;
};
__device__ __forceinline__ PackedItem load_item(const int32_t* items, int i) {
  const int32_t* p = items + (int64_t)i * PK_ITEM;
  PackedItem t;
  t.row0 = __builtin_amdgcn_readfirstlane(p[0]);
  t.rows = __builtin_amdgcn_readfirstlane(p[1]);
  t.pos0 = __builtin_amdgcn_readfirstlane(p[2]);
  t.other0 = __builtin_amdgcn_readfirstlane(p[3]);
  t.other_len = __builtin_amdgcn_readfirstlane(p[4]);
  t.bound = __builtin_amdgcn_readfirstlane(p[5]);
  t.shift = __builtin_amdgcn_readfirstlane(p[6]);
  return t;
}
// Whether the item stays inside the packed rows it names (tables come from lbw_attention_packed_plan;
// one made for other tensors is skipped rather than followed out of them).
__device__ __forceinline__ bool item_fits(const PackedItem& t, int64_t own, int64_t other) {
  return t.row0 >= 0 && t.rows > 0 && t.rows <= PK_BLOCK && (int64_t)t.row0 + t.rows <= own &&
         t.pos0 >= 0 && t.other0 >= 0 && t.other_len >= 0 &&
         (int64_t)t.other0 + t.other_len <= other && t.bound >= 0 && t.bound <= t.other_len;
}

// Workgroup i works on item i / Hq (the costliest first) for head i % Hq, counted with the
// key/value head fastest: with a multiple of 8 of them, every XCD keeps its own key/value heads in L2.
__device__ __forceinline__ void pick_head(uint32_t c, int Hk, int group, int& h, int& kv) {
  kv = c % (uint32_t)Hk;
  h = kv * group + c / (uint32_t)Hk;
}

// A workgroup's item, head and piece. Split items come first, all pieces of the costliest ahead: item,
// piece, head; then the others: item, head.
struct PackedShare {
  int item, head, piece;
  bool split;  // the item may have several pieces
};
__device__ __forceinline__ PackedShare pick_share(const PackedArgs& a, uint32_t b, int heads) {
  const uint32_t cut = (uint32_t)a.n_split * a.smax * heads;
  PackedShare s;
  if (b < cut) {
    const uint32_t r = b % ((uint32_t)a.smax * heads);
    s = {(int)(b / ((uint32_t)a.smax * heads)), (int)(r % heads), (int)(r / heads), true};
  } else {
    s = {a.n_split + (int)((b - cut) / heads), (int)((b - cut) % heads), 0, false};
  }
  return s;
}
__device__ __forceinline__ int pieces_of(const PackedArgs& a, const PackedShare& s, int tiles) {
  if (!s.split) return 1;
  const int n = (tiles + a.piece - 1) / a.piece;
  return n < 1 ? 1 : (n < a.smax ? n : a.smax);
}
// Piece's partial result, `floats` of them for each.
__device__ __forceinline__ float* part_of(const PackedArgs& a, const PackedShare& s, int heads, int piece,
                                          int floats) {
  return a.part + (((int64_t)s.item * heads + s.head) * a.smax + piece) * floats;
}
// 16 accumulator registers x 4 blocks of a wave to and from memory in register order: 16 bytes per
// lane, a wave's kilobytes one after another.
__device__ __forceinline__ void store_acc(float* p, int wave, int lane, const floatx16 (&acc)[4]) {
  floatx4* d = reinterpret_cast<floatx4*>(p) + 1024 * wave + lane;
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const floatx16& y = acc[x >> 2];
    const int e = 4 * (x & 3);
    d[64 * x] = floatx4{y[e], y[e + 1], y[e + 2], y[e + 3]};
  }
}
// ... and one block `db` of them, of wave `wave`'s rows, added up: a joining kernel has a wave for each block, as
// one for all four waits longer (16 rows over 8192 keys x 40/8 heads, forward with join 40 / 32 us; gradient of
// 2048 x 40/8 211 / 190).
__device__ __forceinline__ void add_block(const float* p, int wave, int db, int lane, float f, floatx16& acc) {
  const floatx4* d = reinterpret_cast<const floatx4*>(p) + 1024 * wave + 256 * db + lane;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const floatx4 v = d[64 * x];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[4 * x + e] += f * v[e];
  }
}

// This wave's share of a tile copied HBM -> LDS: rows first .. first + 63 of a sequence of `len`
// rows at `base` (its row 0), row stride `stride_b` bytes; rows past the end copy the last row, so
// a tile never touches another sequence.
struct TileCopy {
  int row0, col0;
  __device__ __forceinline__ void init(int wave, int lane) {
    // copy i fills the wave's 1 KB block i: row row0 + 4 i, chunk (lane % 16) ^ swz(row), whose
    // (row / 4) % 4 part is i, as a wave's four blocks are rows 16 wave ..
    static_assert(PK_NDMA == 4, "four blocks of four rows per wave");
    row0 = 16 * wave + (lane >> 4);
    col0 = ((lane & 15) ^ swz(lane >> 4)) * 16;
  }
  // byte offset of row row0, kept by the caller for a tensor's stride
  __device__ __forceinline__ uint32_t row_offset(int64_t stride_b) const {
    return (uint32_t)row0 * (uint32_t)stride_b;
  }
  // Rows of a whole tile: two vector instructions a copy, the rest is scalar. (With each row's clamp and
  // product taken for every tile, 6 vector instructions and 5 wait states a copy, the forward took 394 us
  // at 4680 + 3600 + 1561 tokens x 40/8 heads.)
  __device__ __forceinline__ void issue(const unsigned char* base, int64_t stride_b, uint32_t off, int first,
                                        int len, uint32_t dst) const {
    const unsigned char* b = base + (int64_t)first * stride_b;
    const int last = len - 1 - first;
    if (last >= BN - 1) {
#pragma unroll
      for (int i = 0; i < PK_NDMA; ++i) dma16(b + 4 * i * stride_b, off + (col0 ^ (i << 4)), dst + 1024 * i);
    } else {
#pragma unroll
      for (int i = 0; i < PK_NDMA; ++i) {
        const int r = row0 + 4 * i < last ? row0 + 4 * i : last;
        dma16(b, (uint32_t)r * (uint32_t)stride_b + (col0 ^ (i << 4)), dst + 1024 * i);
      }
    }
  }
};

// Per-lane LDS byte addresses of a tile's fragments (32-row block 0 at `base`, a multiple of 1 KB).
// The swizzle only exchanges bits 4 to 7 of an address, so the fragments of a tile differ from one
// of them by an exclusive or and a constant: one register each instead of eight.
// Row reads (A operand, d-slice s): row l32, logical chunk 2s + hl.
__device__ __forceinline__ int row_address(int base, int l32, int hl) {
  return base + l32 * PK_ROWB + ((hl ^ swz(l32)) << 4);
}
__device__ __forceinline__ u32x4 read_row(int addr, int s, int at) {
  return lds_read_b128((addr ^ (s << 5)) + at);
}
// Transpose reads for d-block db and row half j: source row 4hl + 8j + s / 4, columns
// 32 db + 16 g + 4 (s % 4) .. +3 (s = lane % 16, g = (lane / 16) % 2); rows 16m further along
// give the lane values k = 16m + 4hl + 8 (e / 4) + e % 4 of the operand's k-group, the order of
// the accumulator registers 8m + e.
__device__ __forceinline__ int tr_address(int base, int lane, int hl) {
  const int s16 = lane & 15, g = (lane >> 4) & 1;
  const int r = 4 * hl + (s16 >> 2), lc = 2 * g + ((s16 & 3) >> 1);
  return base + r * PK_ROWB + ((lc ^ swz(r)) << 4) + 8 * (s16 & 1);
}
__device__ __forceinline__ u32x4 read_tr(int addr, int db, int m, int at) {
  const int x = addr ^ (db << 6);  // (chunk 4 db; rows 8 further: swz's low part changes by 2)
  const u32x2 v0 = lds_read_tr16(x + at + 16 * m * PK_ROWB);
  const u32x2 v1 = lds_read_tr16((x ^ 32) + at + (16 * m + 8) * PK_ROWB);
  return u32x4{v0[0], v0[1], v1[0], v1[1]};
}

// Index within its 32-block of accumulator register r (rows of the product).
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

__device__ __forceinline__ void zero(floatx16& x) {
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = 0.0f;
}

// Registers 8m .. 8m + 7 as a bf16 operand of 8 k-values.
__device__ __forceinline__ u32x4 pack_half(const floatx16& p, int m) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(p[8 * m + 2 * e], p[8 * m + 2 * e + 1]);
  return w;
}

// A wave's [32 rows x 128] result from the transposed accumulators (lane: row l32, d = 32 db +
// 8 g + 4 hl ..) times f, to bf16 rows: through 8 KB of LDS, so that whole rows leave.
template <typename RowPtr>
__device__ __forceinline__ void store_rows(unsigned char* stg, const floatx16 (&acc)[4], float f,
                                           int lane, int rows, RowPtr row_ptr) {
  const int l32 = lane & 31, hl = lane >> 5;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x2 w;
      w[0] = pack_bf16x2(acc[db][4 * g + 0] * f, acc[db][4 * g + 1] * f);
      w[1] = pack_bf16x2(acc[db][4 * g + 2] * f, acc[db][4 * g + 3] * f);
      *reinterpret_cast<u32x2*>(stg + l32 * 256 + (((4 * db + g) ^ (l32 & 15)) << 4) + 8 * hl) = w;
    }
  wave_lds_fence();
  const int rrow = lane >> 4, rch = lane & 15;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int r = 4 * k + rrow;
    const u32x4 v = *reinterpret_cast<const u32x4*>(stg + r * 256 + ((rch ^ (r & 15)) << 4));
    if (r < rows) *reinterpret_cast<u32x4*>(row_ptr(r) + 8 * rch) = v;
  }
}

// One block of it, straight to the rows.
template <typename RowPtr>
__device__ __forceinline__ void store_block(const floatx16& acc, float f, int db, int lane, int rows,
                                            RowPtr row_ptr) {
  const int l32 = lane & 31, hl = lane >> 5;
  if (l32 >= rows) return;
  uint16_t* p = row_ptr(l32) + 32 * db + 4 * hl;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x2 w;
    w[0] = pack_bf16x2(acc[4 * g + 0] * f, acc[4 * g + 1] * f);
    w[1] = pack_bf16x2(acc[4 * g + 2] * f, acc[4 * g + 3] * f);
    *reinterpret_cast<u32x2*>(p + 8 * g) = w;
  }
}

// 32 rows x 128 as a B operand in registers: lane column l32 holds row min(l32, rows - 1),
// d = 16 s + 8 hl .. +7.
__device__ __forceinline__ void load_rows(const uint16_t* base, int64_t stride, int rows, int l32,
                                          int hl, u32x4 (&f)[8]) {
  const int r = l32 < rows ? l32 : rows - 1;
  const uint16_t* p = base + (int64_t)r * stride + 8 * hl;
#pragma unroll
  for (int s = 0; s < 8; ++s) f[s] = *reinterpret_cast<const u32x4*>(p + 16 * s);
}

}  // namespace lbw
