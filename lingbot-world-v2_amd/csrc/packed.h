// Kernel-argument structs and launchers of the operators on packed sequences (internal to the
// library): per-head norm + rotation, packed attention with its gradient, single-token attention.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lbw {

constexpr int kMaxAxes = 4;
constexpr int HN_WAVES = 4;    // per-head norm: waves per workgroup

// One tensor of token rows: element strides of a token and of a head.
struct Rows {
  const uint16_t* p;
  int64_t sl, sh;
};
struct RowsOut {
  uint16_t* p;
  int64_t sl, sh;
};

struct HeadNormArgs {
  int T, Hq, Hk;
  Rows q, k, v;               // v: copied to vo (null: none)
  const void* wq;             // [D] or null (1)
  const void* wk;
  int w32;                    // weights are fp32 (else bf16)
  float eps, inv_d;
  const float2* table;        // [P][npairs] (cos, sin)
  int P, npairs;
  int ax_end[kMaxAxes];       // pair i turns with axis a when ax_end[a - 1] <= i < ax_end[a]
  int naxes, inter;
  const int32_t* pos;         // [T][naxes], row stride pos_sl
  int64_t pos_sl;
  RowsOut qo, ko, vo;         // forward outputs; gradient: dq, dk
  // row form: token t's K and V go to row rows[t] of sequence t (strides kosb, vosb), if in range
  const int32_t* rows;
  int cap;
  int64_t kosb, vosb;
  float q_scale, k_scale;
  int parts;                  // waves that share one token's heads (forward)
  // gradient
  Rows dqo, dko;
  float* part;                // [nwg][D] partial weight gradients
  int nwg, nwg_q;             // workgroups of the gradient; the first nwg_q of them take q
  void* dwq;                  // [D] each, of the weights' type, or null
  void* dwk;
};
hipError_t launch_head_norm(const HeadNormArgs& a, int D, hipStream_t stream);
hipError_t launch_head_norm_bwd(const HeadNormArgs& a, int D, hipStream_t stream);
int head_norm_bwd_workgroups(int T, int cus);

// ---- packed attention
constexpr int PK_BLOCK = 128;       // queries (forward, dQ) or keys (dK, dV) of a work item
constexpr int PK_ITEM = 8;          // int32 fields of an item
// Query item: {first packed query row, rows, their index in the sequence, sequence's first packed
// key row, its keys, keys that the item's last row sees, shift, 0}: query i of a sequence sees keys
// j < k_len with j <= i + shift (causal: k_len - q_len; full: k_len).
// Key item: {first packed key row, rows, their index in the sequence, sequence's first packed
// query row, its queries, first query that sees any of the rows, shift, 0}.
struct PackedArgs {
  Rows q, k, v;
  RowsOut out;                 // forward
  float* lse;                  // [Hq][Tq] natural log; null: not wanted
  int64_t Tq, Tk;              // packed rows of q and of k, v
  int Hq, Hk;
  float scale, scale_log2;
  const int32_t* q_items;
  const int32_t* k_items;
  int n_q_items, n_k_items;
  // The first n_split items are cut into pieces of about `piece` tiles, at most smax, when they are
  // longer; a piece leaves fp32 partial results in `part`, which a second kernel joins in their order.
  int n_split, smax, piece;
  float* part;
  // gradient
  bool halves;                 // dK, dV: 64 keys per workgroup
  Rows o, dout;
  float* ndelta;               // [Hq][Tq]: -sum_d dout out
  float* nlse;                 // [Hq][Tq]: -lse / scale, -inf for a query that sees no key
  RowsOut dq, dk, dv;
};
struct PackedSplit {
  int n_split, smax, piece;
};
// Floats of a piece's partial result: forward (O, m, l), dQ, dK + dV of 128 rows x 128.
constexpr int PK_PART_FWD = PK_BLOCK * 128 + 2 * PK_BLOCK, PK_PART_DQ = PK_BLOCK * 128,
              PK_PART_DKV = 2 * PK_BLOCK * 128;
hipError_t launch_packed_fwd(const PackedArgs& a, hipStream_t stream);
hipError_t launch_packed_dq(const PackedArgs& a, hipStream_t stream);
hipError_t launch_packed_dkv(const PackedArgs& a, hipStream_t stream);

// ---- single-token attention over per-sequence caches
struct DecodeArgs {
  Rows q;                      // [B, Hq, D]: sl is the batch stride
  const uint16_t* k;           // [B, S, Hk, D]
  const uint16_t* v;
  int64_t ksb, ksl, ksh, vsb, vsl, vsh;
  const int32_t* lens;         // [B]
  RowsOut out;                 // [B, Hq, D]
  int B, Hq, Hk, S;
  float scale, scale_log2;
  int pieces;                  // 0: a workgroup per sequence; J: a key/value head's keys of the whole
                               // batch in J equal pieces
  float* part;                 // pieces: [Hq][pieces + B][D] partial O, then m and l, [Hq][pieces + B] each
};
hipError_t launch_decode(const DecodeArgs& a, hipStream_t stream);
int decode_pieces(int64_t B, int Hq, int Hk, int64_t S, int num_splits, int cus);

}  // namespace lbw
