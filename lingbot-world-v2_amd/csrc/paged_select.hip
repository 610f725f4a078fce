// The pages of a paged cache that a query token should look at (gfx950).
//
//   score(b, g, page) = max over the query heads h of key/value head g of
//                       sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d
//
// with the page's bounds lo <= k <= hi of every key component: no key of the page scores higher. Chosen are the first
// and the last pages of a sequence, then those of the highest scores (ties: the lower page), in ascending order.
//
// Scores are sums in 64 bits: a product of two bf16 values has 16 bits, so such a sum is exact unless its terms span
// more than 2^30, and the choice does not hang on the order of additions. A score is bound by reading the bounds, 512
// bytes per page and head against 16 KB and more of the page's keys; the choice by its rounds of counting.
//
// A wave scores four pages at a time: 16 lanes a page, 8 components each, with q's positive and negative parts in
// registers. The second kernel has a workgroup per sequence and key/value head: it narrows the range of scores that
// holds the last chosen one, 1024 equal bins at a time, until the choice is settled (a few rounds).

#include "capi_util.h"
#include "head_rows.h"
#include "paged.h"

namespace lbw {
namespace {

constexpr int SEL_D = 128;
constexpr int SC_PAGES = 32;      // pages of a workgroup of the score kernel
constexpr int SC_G = 5;           // query heads at a time, at most (64 registers of q each two)
constexpr int TOP_T = 1024;       // threads of the choice, and bins
constexpr int TOP_U = 4;          // scores per thread in registers
constexpr uint64_t INF_IMAGE = 0xfff0000000000000ull;

// Order-preserving image of a score: -0 as 0, NaN as infinity.
__device__ __forceinline__ uint64_t image(double x) {
  if (x != x) return INF_IMAGE;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : u | (1ull << 63);
}

// x plus the value of another lane of its row of 16, by a DPP pattern.
template <int CTRL>
__device__ __forceinline__ double add_dpp(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return x + __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
// Sum over 16 lanes, in all of them: neighbours, pairs, then mirrored halves and rows.
__device__ __forceinline__ double row_sum(double x) {
  x = add_dpp<0xb1>(x);   // quad_perm [1, 0, 3, 2]
  x = add_dpp<0x4e>(x);   // quad_perm [2, 3, 0, 1]
  x = add_dpp<0x141>(x);  // row_half_mirror
  return add_dpp<0x140>(x);  // row_mirror
}

__device__ __forceinline__ int pages_of(const SelectArgs& a, int b) {
  const int64_t cap = (int64_t)a.pt.width << a.pt.shift;
  int64_t n = a.lens[b];
  n = n < 0 ? 0 : (n > cap ? cap : n);
  return __builtin_amdgcn_readfirstlane((int)((n + (1 << a.pt.shift) - 1) >> a.pt.shift));
}

template <int G>
__global__ void __launch_bounds__(256) select_score_kernel(const SelectArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = (uint32_t)((a.pt.width + SC_PAGES - 1) / SC_PAGES);
  const int chunk = blockIdx.x % chunks, kv = (blockIdx.x / chunks) % (uint32_t)a.Hk,
            b = blockIdx.x / chunks / (uint32_t)a.Hk;
  const int n = pages_of(a, b);
  if (n <= a.count || chunk * SC_PAGES >= n) return;  // (all pages are chosen, or none is here)
  const int group = a.Hq / a.Hk, e0 = 8 * (lane & 15), sub = lane >> 4;
  const int32_t* const table = a.pt.p + b * a.pt.sb;
  uint64_t* const score = a.score + ((int64_t)b * a.Hk + kv) * a.pt.width;
  for (int h0 = 0; h0 < group; h0 += G) {
    double up[G][8], down[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float f[8];
      const int h = h0 + g < group ? h0 + g : group - 1;  // (past the last head: it once more)
      unpack8(load16(a.q.p + b * a.q.sl + (int64_t)(kv * group + h) * a.q.sh + e0), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // (a NaN stays in one of the two)
        up[g][j] = f[j] < 0.0f ? 0.0 : (double)f[j];
        down[g][j] = f[j] < 0.0f ? (double)f[j] : 0.0;
      }
    }
#pragma unroll
    for (int i = 0; i < SC_PAGES / 16; ++i) {
      const int page = chunk * SC_PAGES + 16 * i + 4 * wave + sub;
      // (pages past the last are scored too, as page 0, and not written)
      int at = page < n ? page_at(table, a.pt.width, a.pt.shift, a.pt.pages, (int64_t)page << a.pt.shift) : 0;
      const bool bad = at < 0;
      at = bad ? 0 : at;
      const uint16_t* p = a.bounds + ((int64_t)at * a.Hk + kv) * 2 * SEL_D + e0;
      float lo[8], hi[8];
      unpack8(load16(p), lo);
      unpack8(load16(p + SEL_D), hi);
      double x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double l = lo[j], h = hi[j];
#pragma unroll
        for (int g = 0; g < G; ++g) x[g] = __builtin_fma(down[g][j], l, __builtin_fma(up[g][j], h, x[g]));
      }
      uint64_t best = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint64_t u = image(row_sum(x[g]));
        best = u > best ? u : best;
      }
      if (bad) best = INF_IMAGE;
      if (page < n && (lane & 15) == 0) {
        if (h0 > 0 && score[page] > best) best = score[page];
        score[page] = best;
      }
    }
  }
}

// Reductions over a workgroup of 16 waves.
template <typename F>
__device__ __forceinline__ uint64_t reduce64(uint64_t x, F f, uint64_t* red, int lane, int wave) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = f(x, (uint64_t)__shfl_xor((unsigned long long)x, o));
  __syncthreads();
  if (lane == 0) red[wave] = x;
  __syncthreads();
  uint64_t y = red[0];
#pragma unroll
  for (int w = 1; w < TOP_T / 64; ++w) y = f(y, red[w]);
  return y;
}

__global__ void __launch_bounds__(TOP_T) select_top_kernel(const SelectArgs a) {
  __shared__ uint32_t hist[TOP_T], sums[TOP_T / 64][2];
  __shared__ uint64_t red[TOP_T / 64];
  __shared__ uint32_t found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv = blockIdx.x % (uint32_t)a.Hk, b = blockIdx.x / (uint32_t)a.Hk;
  const int n = pages_of(a, b);
  int32_t* const sel = a.sel + ((int64_t)b * a.Hk + kv) * a.count;
  if (n <= a.count) {
    for (int i = tid; i < a.count; i += TOP_T) sel[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* const score = a.score + ((int64_t)b * a.Hk + kv) * a.pt.width;
  auto kept = [&](int i) { return i < a.first || i >= n - a.last; };
  uint64_t mine[TOP_U];
#pragma unroll
  for (int j = 0; j < TOP_U; ++j) mine[j] = j * TOP_T + tid < n ? score[j * TOP_T + tid] : 0;
  // f(score) of every page that is not kept anyway
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < TOP_U; ++j) {
      const int i = j * TOP_T + tid;
      if (i < n && !kept(i)) f(mine[j]);
    }
    for (int i = TOP_U * TOP_T + tid; i < n; i += TOP_T)
      if (!kept(i)) f(score[i]);
  };
  uint32_t need = (uint32_t)(a.count - a.first - a.last);  // (n > count: first and last do not meet)
  uint64_t over = ~0ull;  // chosen: scores above this, and `need` of those that equal it
  if (need > 0) {
    uint64_t lo = ~0ull, hi = 0;
    each([&](uint64_t u) {
      lo = u < lo ? u : lo;
      hi = u > hi ? u : hi;
    });
    lo = reduce64(lo, [](uint64_t x, uint64_t y) { return x < y ? x : y; }, red, lane, wave);
    hi = reduce64(hi, [](uint64_t x, uint64_t y) { return x > y ? x : y; }, red, lane, wave);
    // the last chosen score is in [lo, hi], the need-th highest of those there
    while (true) {
      if (lo == hi) {
        over = lo;
        break;
      }
      const int bits = 64 - __clzll((unsigned long long)(hi - lo)), shift = bits > 10 ? bits - 10 : 0;
      hist[tid] = 0;
      __syncthreads();
      each([&](uint64_t u) {
        if (u >= lo && u <= hi) atomicAdd(&hist[(u - lo) >> shift], 1u);
      });
      __syncthreads();
      // bin tid from the top: how many scores are in it and in those above it
      const uint32_t own = hist[TOP_T - 1 - tid];
      uint32_t sum = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(sum, o);
        if (lane >= o) sum += y;
      }
      if (lane == 63) sums[wave][0] = sum;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TOP_T / 64 - 1; ++w) sum += w < wave ? sums[w][0] : 0;
      if (sum >= need && sum - own < need) {  // one thread: counts reach `need` once
        found[0] = TOP_T - 1 - tid;
        found[1] = own;
        found[2] = need - (sum - own);
      }
      __syncthreads();
      const uint64_t l = lo + ((uint64_t)found[0] << shift), h = l + ((1ull << shift) - 1);
      need = found[2];
      const bool all = need == found[1];
      lo = l;
      hi = h < hi ? h : hi;
      if (all) {  // every score of the bin
        over = lo - 1;
        need = 0;
        break;
      }
      __syncthreads();  // found is read
    }
  }
  // in ascending order: kept pages and scores above come first-come, of equal ones the first `need`
  uint32_t above0 = 0, equal0 = 0;
  const uint64_t before = ((uint64_t)1 << lane) - 1;
  auto put = [&](int i, uint64_t u) {
    const bool is_kept = i < n && kept(i);
    const bool above = is_kept || (i < n && u > over), equal = i < n && !is_kept && u == over;
    const uint64_t ma = __ballot(above), me = __ballot(equal);
    __syncthreads();  // the last sums are read
    if (lane == 0) {
      sums[wave][0] = __popcll(ma);
      sums[wave][1] = __popcll(me);
    }
    __syncthreads();
    uint32_t na = above0 + __popcll(ma & before), ne = equal0 + __popcll(me & before);
#pragma unroll
    for (int w = 0; w < TOP_T / 64; ++w) {
      na += w < wave ? sums[w][0] : 0;
      ne += w < wave ? sums[w][1] : 0;
      above0 += sums[w][0];
      equal0 += sums[w][1];
    }
    if (above || (equal && ne < need)) sel[na + (ne < need ? ne : need)] = i;
  };
#pragma unroll
  for (int j = 0; j < TOP_U; ++j)
    if (j * TOP_T < n) put(j * TOP_T + tid, mine[j]);
  for (int i0 = TOP_U * TOP_T; i0 < n; i0 += TOP_T) put(i0 + tid, i0 + tid < n ? score[i0 + tid] : 0);
}

template <int G>
void score(const SelectArgs& a, hipStream_t stream) {
  const int64_t chunks = (a.pt.width + SC_PAGES - 1) / SC_PAGES;
  hipLaunchKernelGGL(select_score_kernel<G>, dim3((uint32_t)(chunks * a.Hk * a.B)), dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_select(const SelectArgs& a, hipStream_t stream) {
  if (a.pt.width > a.count) {  // (else every page is chosen)
    // a group's heads in equal turns of five at most
    const int group = a.Hq / a.Hk, turns = (group + SC_G - 1) / SC_G;
    switch ((group + turns - 1) / turns) {
      case 1: score<1>(a, stream); break;
      case 2: score<2>(a, stream); break;
      case 3: score<3>(a, stream); break;
      case 4: score<4>(a, stream); break;
      default: score<5>(a, stream); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(select_top_kernel, dim3((uint32_t)((int64_t)a.B * a.Hk)), dim3(TOP_T), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
