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
// registers. A second kernel has a workgroup per sequence and key/value head: it narrows the range of scores that
// holds the last chosen one, 1024 equal bins at a time, until no more than 256 are left (one round mostly), whose ranks
// are counted one against another. Few pages: one kernel for both. Eight sequences of up to 1463 pages x 40/8 heads 16 +
// 8 us (their bounds take 7 at the rate of a large copy, the 64-bit sums 8), one of 732 pages 4.7 + 6.7.

#include "capi_util.h"
#include "head_rows.h"
#include "paged.h"
#include "score_range.h"

namespace lbw {
namespace {

constexpr int SEL_D = 128;
constexpr int SC_G = 5;           // query heads at a time, at most (64 registers of q each two)
constexpr int TOP_T = 256;        // threads of the choice
constexpr int ONE_T = 512;        // threads of the kernel that scores and chooses
constexpr int ONE_PAGES = 256;    // scores that it keeps
constexpr int BINS = SCORE_BINS;
constexpr uint64_t INF_IMAGE = 0xfff0000000000000ull;

// Order-preserving image of a score that is not NaN, -0 as 0; never 0. (NaN counts as infinity.)
__device__ __forceinline__ uint64_t image(double x) {
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

// Scores of a sequence's pages from .. from + most - 1 for one key/value head, four a wave at a time, unless all of its n
// pages are chosen (returns n either way); `put(page, score, first)`: the higher of it and what is there, unless it is
// the first.
template <int G, typename Put>
__device__ __forceinline__ int score_pages(const SelectArgs& a, int b, int kv, int from, int most, int lane, int wave,
                                           int waves, Put put) {
  const int group = a.Hq / a.Hk, e0 = 8 * (lane & 15), step = 4 * waves, first = from + 4 * wave + (lane >> 4);
  const int32_t* const table = a.pt.p + b * a.pt.sb;
  int n = 0, end = 0;
  for (int h0 = 0; h0 < group; h0 += G) {
    // the queries and the first page's entry are on their way together with the length
    u32x4 raw[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int h = h0 + g < group ? h0 + g : group - 1;  // (past the last head: it once more)
      raw[g] = load16(a.q.p + b * a.q.sl + (int64_t)(kv * group + h) * a.q.sh + e0);
    }
    int page = first;
    int32_t entry = page < a.pt.width ? table[page] : 0;
    if (h0 == 0) {
      n = pages_of(a, b);
      if (n <= a.count || from >= n) return n;
      end = n < from + most ? n : from + most;
    }
    // a page's bounds are fetched while the one before is summed, its entry while the one before that is
    u32x4 lw, hw;
    bool bad = false;
    auto fetch = [&](int next) {
      int at = page_of_entry(entry, a.pt.pages);
      bad = at < 0;
      at = bad ? 0 : at;  // (pages past the last are scored too, as page 0 or any, and not written)
      const uint16_t* p = a.bounds + ((int64_t)at * a.Hk + kv) * 2 * SEL_D + e0;
      lw = load16(p);
      hw = load16(p + SEL_D);
      entry = next < end ? table[next] : 0;
    };
    fetch(page + step);
    double up[G][8], down[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float f[8];
      unpack8(raw[g], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // (a NaN stays in one of the two)
        up[g][j] = f[j] < 0.0f ? 0.0 : (double)f[j];
        down[g][j] = f[j] < 0.0f ? (double)f[j] : 0.0;
      }
    }
    for (; __any(page < end); page += step) {
      float lo[8], hi[8];
      unpack8(lw, lo);
      unpack8(hw, hi);
      const bool is_bad = bad;
      fetch(page + 2 * step);
      double x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double l = lo[j], h = hi[j];
#pragma unroll
        for (int g = 0; g < G; ++g) x[g] = __builtin_fma(down[g][j], l, __builtin_fma(up[g][j], h, x[g]));
      }
      double best = -INFINITY;
      bool nan = is_bad;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const double y = row_sum(x[g]);
        nan |= y != y;
        best = fmax(best, y);
      }
      const uint64_t s = nan ? INF_IMAGE : image(best);
      if (page < end && (lane & 15) == 0) put(page, s, h0 == 0);
    }
  }
  return n;
}

template <int G>
__global__ void __launch_bounds__(256) select_score_kernel(const SelectArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = (uint32_t)((a.pt.width + a.chunk - 1) / a.chunk), unit = blockIdx.x / (uint32_t)a.Hk;
  // (another chunk first in each sequence: the last ones, of few pages or none, would often meet on one XCD; 64 sequences
  // of up to 98 pages x 40/8 heads 22.4 to 18.5 us, 16 of 1463 x 64/8 48.1 to 43.8)
  const int kv = blockIdx.x % (uint32_t)a.Hk, b = unit / chunks, chunk = (unit % chunks + (uint32_t)b) % chunks;
  uint64_t* const score = a.score + ((int64_t)b * a.Hk + kv) * a.pt.width;
  score_pages<G>(a, b, kv, chunk * a.chunk, a.chunk, lane, wave, 4, [&](int page, uint64_t best, bool first) {
    if (!first && score[page] > best) best = score[page];
    score[page] = best;
  });
}

// The choice among n > count pages by their scores, by T threads.
template <int T>
__device__ __forceinline__ void choose(const SelectArgs& a, int n, const uint64_t* score, int32_t* sel) {
  constexpr int TOP_W = T / 64;
  constexpr int TOP_U = 64 / TOP_W;  // scores per thread in registers
  __shared__ uint32_t hist[BINS], sums[TOP_W], counts[TOP_U * TOP_W][2];
  __shared__ uint64_t range[TOP_W][2], cand[T], border;
  __shared__ int32_t place[T];
  __shared__ uint32_t found[3], collected;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto kept = [&](int i) { return i < a.first || i >= n - a.last; };
  // 0 for a page that is kept anyway, or is none
  auto score_of = [&](int i) { return i < n && !kept(i) ? score[i] : 0; };
  // page j * T + tid in mine[j]; those past TOP_U * T are read anew each time
  uint64_t mine[TOP_U];
#pragma unroll
  for (int j = 0; j < TOP_U; ++j) mine[j] = j * T < n ? score_of(j * T + tid) : 0;
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < TOP_U; ++j) {
      if (j * T >= n) break;
      f(mine[j], j * T + tid);
    }
    for (int i = TOP_U * T + tid; i < n; i += T) f(score_of(i), i);
  };
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < BINS / T; ++i) hist[i * T + tid] = 0;
  };
  uint32_t need = (uint32_t)(a.count - a.first - a.last);  // (n > count: first and last do not meet)
  uint64_t over = ~0ull;  // chosen: scores above this, and the first `need` of those that equal it
  if (need > 0) {
    uint64_t lo = ~0ull, hi = 0;
    each([&](uint64_t u, int) {
      lo = u - 1 < lo ? u - 1 : lo;  // (0 becomes the largest)
      hi = u > hi ? u : hi;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t x = (uint64_t)__shfl_xor((unsigned long long)lo, o);
      const uint64_t y = (uint64_t)__shfl_xor((unsigned long long)hi, o);
      lo = x < lo ? x : lo;
      hi = y > hi ? y : hi;
    }
    if (lane == 0) {
      range[wave][0] = lo;
      range[wave][1] = hi;
    }
    if (tid == 0) collected = 0;
    clear();
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TOP_W; ++w) {
      lo = range[w][0] < lo ? range[w][0] : lo;
      hi = range[w][1] > hi ? range[w][1] : hi;
    }
    ScoreRange r = {lo + 1, hi};
    // the last chosen score is in the range, the need-th highest of those there
    while (true) {
      if (r.lo == r.hi) {
        over = r.lo;
        break;
      }
      const int shift = bin_shift(r);
      each([&](uint64_t u, int) {
        if (in_range(r, u)) atomicAdd(&hist[bin_of(r, shift, u)], 1u);
      });
      __syncthreads();
      // four bins a thread, from the top: how many scores are in them and in those above
      constexpr int BPT = BINS / T;
      uint32_t own[BPT], sum = 0;
#pragma unroll
      for (int i = 0; i < BPT; ++i) sum += own[i] = hist[BINS - 1 - (tid * BPT + i)];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 63) sums[wave] = upto;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TOP_W - 1; ++w) upto += w < wave ? sums[w] : 0;
      upto -= sum;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (upto < need && upto + own[i] >= need) {  // one bin: counts reach `need` once
          found[0] = BINS - 1 - (tid * BPT + i);
          found[1] = own[i];
          found[2] = need - upto;
        }
        upto += own[i];
      }
      clear();
      __syncthreads();
      r = bin_range(r, shift, (int)found[0]);
      need = found[2];
      const uint32_t in_bin = found[1];
      if (need == in_bin) {  // every score of the bin
        over = r.lo - 1;
        need = 0;
        break;
      }
      if (in_bin <= T) {
        each([&](uint64_t u, int i) {
          if (in_range(r, u)) {
            const uint32_t at = atomicAdd(&collected, 1u);
            cand[at] = u;
            place[at] = i;
          }
        });
        __syncthreads();
        if (tid < (int)in_bin) {  // (their order differs from run to run, their ranks do not)
          const uint64_t u = cand[tid];
          const int32_t i = place[tid];
          uint32_t above = 0, rank = 0;
          for (uint32_t j = 0; j < in_bin; ++j) {
            above += cand[j] > u;
            rank += cand[j] > u || (cand[j] == u && place[j] < i);
          }
          if (rank == need - 1) {
            border = u;
            found[2] = need - above;
          }
        }
        __syncthreads();
        over = border;
        need = found[2];
        break;
      }
      __syncthreads();  // found is read
    }
  }
  // in ascending order: kept pages and scores above, of equal ones the first `need`
  const uint64_t before = ((uint64_t)1 << lane) - 1;
  uint32_t above0 = 0, equal0 = 0;
  for (int base = 0; base < n; base += TOP_U * T) {
    // a page's: bit 16 above, bit 17 equal, and how many above (bits 0 ..) and equal ones (bits 8 ..) the wave's lower
    // lanes hold
    uint32_t turn[TOP_U];
#pragma unroll
    for (int j = 0; j < TOP_U; ++j) {
      turn[j] = 0;
      if (base + j * T >= n) continue;
      const int i = base + j * T + tid;
      const uint64_t u = base == 0 ? mine[j] : score_of(i);
      const bool above = (i < n && kept(i)) || u > over, equal = u == over;
      const uint64_t ma = __ballot(above), me = __ballot(equal);
      turn[j] = (uint32_t)__popcll(ma & before) | (uint32_t)__popcll(me & before) << 8 | (above ? 1u << 16 : 0) |
                (equal ? 1u << 17 : 0);
      if (lane == 0) {
        counts[j * TOP_W + wave][0] = __popcll(ma);
        counts[j * TOP_W + wave][1] = __popcll(me);
      }
    }
    __syncthreads();
    // lane x: how many are in the first x + 1 of the waves' turns
    static_assert(TOP_U * TOP_W == 64, "a lane for each turn of each wave");
    const bool there = base + (lane / TOP_W) * T < n;
    const uint32_t na = there ? counts[lane][0] : 0, ne = there ? counts[lane][1] : 0;
    uint32_t sa = na, se = ne;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(sa, o), y = __shfl_up(se, o);
      if (lane >= o) {
        sa += x;
        se += y;
      }
    }
#pragma unroll
    for (int j = 0; j < TOP_U; ++j) {
      if (base + j * T >= n) continue;
      const int x = j * TOP_W + wave;
      const uint32_t pa = above0 + __builtin_amdgcn_readlane(sa - na, x) + (turn[j] & 255);
      const uint32_t pe = equal0 + __builtin_amdgcn_readlane(se - ne, x) + (turn[j] >> 8 & 255);
      const uint32_t at = pa + (pe < need ? pe : need);
      // (the list's end is asked for all the same: what is behind it is another list)
      if (((turn[j] >> 16 & 1) || ((turn[j] >> 17) && pe < need)) && at < (uint32_t)a.count) sel[at] = base + j * T + tid;
    }
    above0 += __shfl(sa, 63);
    equal0 += __shfl(se, 63);
    __syncthreads();  // the counts are read
  }
}

// All of a sequence's pages, where there are no more than `count`.
template <int T>
__device__ __forceinline__ bool chose_all(const SelectArgs& a, int n, int32_t* sel) {
  if (n > a.count) return false;
  for (int i = threadIdx.x; i < a.count; i += T) sel[i] = i < n ? i : -1;
  return true;
}

__global__ void __launch_bounds__(TOP_T) select_top_kernel(const SelectArgs a) {
  const int kv = blockIdx.x % (uint32_t)a.Hk, b = blockIdx.x / (uint32_t)a.Hk;
  const int n = pages_of(a, b);
  int32_t* const sel = a.sel + ((int64_t)b * a.Hk + kv) * a.count;
  if (!chose_all<TOP_T>(a, n, sel)) choose<TOP_T>(a, n, a.score + ((int64_t)b * a.Hk + kv) * a.pt.width, sel);
}

// Both for a sequence and key/value head of few pages, whose scores stay in LDS.
template <int G>
__global__ void __launch_bounds__(ONE_T) select_one_kernel(const SelectArgs a) {
  __shared__ uint64_t score[ONE_PAGES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv = blockIdx.x % (uint32_t)a.Hk, b = blockIdx.x / (uint32_t)a.Hk;
  int32_t* const sel = a.sel + ((int64_t)b * a.Hk + kv) * a.count;
  const int n = score_pages<G>(a, b, kv, 0, ONE_PAGES, lane, wave, ONE_T / 64, [&](int page, uint64_t best, bool first) {
    score[page] = first || best > score[page] ? best : score[page];
  });
  if (chose_all<ONE_T>(a, n, sel)) return;
  __syncthreads();
  choose<ONE_T>(a, n, score, sel);
}

template <int G>
void score(const SelectArgs& a, hipStream_t stream) {
  if (a.chunk == 0) {
    hipLaunchKernelGGL(select_one_kernel<G>, dim3((uint32_t)((int64_t)a.B * a.Hk)), dim3(ONE_T), 0, stream, a);
    return;
  }
  const int64_t chunks = (a.pt.width + a.chunk - 1) / a.chunk;
  hipLaunchKernelGGL(select_score_kernel<G>, dim3((uint32_t)(chunks * a.Hk * a.B)), dim3(256), 0, stream, a);
}

}  // namespace

// One kernel while a workgroup for each sequence and key/value head has little to score and a CU of its own. Two kernels
// / one, tables of 20, 64, 128 and 192 pages, us: eight sequences x 40/8 heads 9.7 / 7.7, 9.7 / 8.7, 9.9 / 10.6, 10.9 / 12.3; x
// 12/4 9.6 / 7.1, 9.6 / 8.0, 9.7 / 9.3, 9.6 / 10.5; x 12/12 9.7 / 6.9, 9.7 / 7.4, 9.6 / 8.4, 9.7 / 9.2 (256: 9.8 / 10.4); x 64/8
// 10.8 / 9.2, 11.4 / 10.8, 11.4 / 14.0, 13.2 / 17.0; 64 sequences x 12/4 9.5 / 7.4, 9.8 / 8.2, 11.7 / 9.5, 13.4 / 10.8, x 40/8
// (512 workgroups) 10.8 / 14.0, 14.5 / 15.6, 17.4 / 19.0, 21.4 / 22.8.
void plan_select(SelectArgs* a, int cus) {
  const int64_t rows = (int64_t)a->B * a->Hk, width = a->pt.width;
  a->chunk = 0;
  if (width <= ONE_PAGES && rows <= cus && (a->Hq / a->Hk + 2) * width <= 700) return;
  // pages of a workgroup: 32, more once that gives eight workgroups a CU (each turns its q into 64 bits first)
  a->chunk = 32;
  while (a->chunk < 256 && rows * width > (int64_t)8 * cus * a->chunk) a->chunk *= 2;
}

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
    if (e != hipSuccess || a.chunk == 0) return e;
  }
  hipLaunchKernelGGL(select_top_kernel, dim3((uint32_t)((int64_t)a.B * a.Hk)), dim3(TOP_T), 0, stream, a);
  return hipGetLastError();
}

}  // namespace lbw
