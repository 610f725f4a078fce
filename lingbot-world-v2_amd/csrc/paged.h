// Kernel-argument structs and launchers of the operators over a paged key/value cache (internal to the
// library): appending tokens, choosing pages, attention of one query token per sequence.
//
// A page holds 2^shift consecutive tokens of one sequence; entry j of a sequence's row of the page table is the
// page of its tokens j 2^shift ... An entry outside the cache never leads a kernel outside it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "packed.h"
#include "page_lookup.h"

namespace lbw {

constexpr int PG_MIN_SHIFT = 4, PG_MAX_SHIFT = 10;  // pages of 16 to 1024 tokens

// K or V of the cache: element strides of a page, of a token within it, and of a head.
struct PageRows {
  uint16_t* p;
  int64_t sp, sl, sh;
};
struct PageTable {
  const int32_t* p;
  int64_t sb;                 // elements between two sequences' rows
  int width;                  // entries of a row
  int shift;
  int pages;                  // of the cache
};

struct AppendArgs {
  int T, B, Hq, Hk;
  Rows q, k, v;
  RowsOut qo;
  const void* wq;             // [D] or null (1)
  const void* wk;
  int w32, norm;
  float eps, inv_d;
  const float2* table;        // rotation, as in HeadNormArgs
  int P, npairs;
  int ax_end[kMaxAxes];
  int naxes, inter;
  const int32_t* pos;         // null: a token's row in its sequence (one axis)
  int64_t pos_sl;
  const int32_t* starts;      // [B + 1] first token of each sequence; null: token t is sequence t's
  const int32_t* lens;        // [B] rows that a sequence has so far
  PageTable pt;
  PageRows kp, vp;
  uint16_t* bounds;           // [pages][Hk][2][D] smallest and largest values, or null
  float q_scale, k_scale;
  int parts;                  // waves that share one token's heads
  int page_wgs, page_heads;   // workgroups that look after pages' new keys, and the heads of each
  int page_slots;             // they are told apart by pages (else by tokens)
};
hipError_t launch_append(const AppendArgs& a, int D, hipStream_t stream);

struct PagedAttnArgs {
  Rows q;                     // [B, Hq, D]: sl is the batch stride
  PageRows k, v;
  PageTable pt;
  const int32_t* lens;        // [B]
  const int32_t* sel;         // [B][Hk][n_sel] entries of the table to attend to, up to the first negative one;
  int n_sel;                  // null: all
  RowsOut out;                // [B, Hq, D]
  int B, Hq, Hk, group;       // group: Hq / Hk
  float scale, scale_log2;
  // own keys: the whole batch's in `pieces` equal pieces per key/value head, or (pieces 0) each sequence's in
  // `splits`
  int pieces, splits;
  // common prefix: keys that come before every sequence's own, in p_splits pieces (0: none)
  const int32_t* p_table;
  int p_width;
  const int32_t* p_len;       // [1] or null
  int64_t p_max;              // at most so many keys
  int p_splits, p_block;      // p_block: query rows of a workgroup
  int p_inline;               // every sequence walks the prefix itself, before its own keys (p_splits 0)
  // partial results: own parts then the prefix's, [Hq][rows][D] each, then m and l of all of them
  float* part;
};
// Rows of partial results per query head: own parts and the prefix's.
__host__ __device__ inline int64_t own_rows(const PagedAttnArgs& a) {
  return a.pieces > 0 ? (int64_t)a.pieces + a.B : (int64_t)a.B * a.splits;
}
__host__ __device__ inline int64_t all_rows(const PagedAttnArgs& a) { return own_rows(a) + (int64_t)a.B * a.p_splits; }
// Whether results go through partial ones.
__host__ __device__ inline bool has_parts(const PagedAttnArgs& a) {
  return a.pieces > 0 || a.splits > 1 || a.p_splits > 0;
}
// Workgroups per key/value head: of the prefix, and of own keys (32 query rows each).
inline int64_t prefix_units(const PagedAttnArgs& a) {
  return a.p_splits > 0 ? a.p_splits * (((int64_t)a.B * a.group + a.p_block - 1) / a.p_block) : 0;
}
inline int64_t own_units(const PagedAttnArgs& a) {
  return (a.pieces > 0 ? (int64_t)a.pieces : (int64_t)a.B * a.splits) * ((a.group + 31) / 32);
}
inline int64_t workgroups(const PagedAttnArgs& a) { return (prefix_units(a) + own_units(a)) * a.Hk; }
hipError_t launch_paged(const PagedAttnArgs& a, hipStream_t stream);
void plan_paged(PagedAttnArgs* a, int num_splits, int cus);

struct SelectArgs {
  Rows q;
  const uint16_t* bounds;     // [pages][Hk][2][D]
  PageTable pt;
  const int32_t* lens;
  int B, Hq, Hk, count, first, last;
  int chunk;                  // pages that a workgroup of the score kernel takes; 0: one kernel does all
  uint64_t* score;            // [B][Hk][width] order-preserving images of the scores
  int32_t* sel;               // [B][Hk][count]
};
void plan_select(SelectArgs* a, int cus);
hipError_t launch_select(const SelectArgs& a, hipStream_t stream);

}  // namespace lbw
