// Tiles of a batch's sequences laid end to end (single-token attention): lengths are on the device, so a wave
// counts them there, 64 sequences at a time. tiles(b) gives those of sequence b of B.
#pragma once

#include "common.h"

namespace lbw {

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ int64_t scalar64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// Tiles of all sequences together and, with `upto`, of those before it.
template <typename Tiles>
__device__ __forceinline__ void count_tiles_of(int B, Tiles tiles, int lane, int upto, int64_t& all,
                                               int64_t& before) {
  int64_t x = 0, y = 0;
  for (int b = lane; b < B; b += 64) {
    const int n = tiles(b);
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
template <typename Tiles>
__device__ __forceinline__ int find_sequence(int B, Tiles tiles, int lane, int64_t t, int64_t& before) {
  int64_t base = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int n = b0 + lane < B ? tiles(b0 + lane) : 0;
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
  return B;
}

}  // namespace lbw
