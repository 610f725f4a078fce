// The range of page scores that holds the last chosen one, narrowed by equal bins: the arithmetic of the choice among
// pages, on the device and in the host's tests. Plain C++.
#pragma once

#include <stdint.h>

#include "page_lookup.h"

namespace lbw {

constexpr int SCORE_BINS = 1024;

// Scores lo .. hi (lo <= hi), as order-preserving 64-bit images: those of infinity lie within 2^52 of the largest
// number, so no bound is formed by adding to a score.
struct ScoreRange {
  uint64_t lo, hi;
};
LBW_LOOKUP bool in_range(const ScoreRange& r, uint64_t u) { return u >= r.lo && u <= r.hi; }
// A bin holds 2^shift scores, of a range of more than one.
LBW_LOOKUP int bin_shift(const ScoreRange& r) {
  const int bits = 64 - __builtin_clzll((unsigned long long)(r.hi - r.lo));
  return bits > 10 ? bits - 10 : 0;
}
LBW_LOOKUP int bin_of(const ScoreRange& r, int shift, uint64_t u) { return (int)((u - r.lo) >> shift); }
// The part of the range that a bin covers (one that holds a score of the range).
LBW_LOOKUP ScoreRange bin_range(const ScoreRange& r, int shift, int bin) {
  const uint64_t lo = r.lo + ((uint64_t)bin << shift), rest = r.hi - lo, most = ((uint64_t)1 << shift) - 1;
  return ScoreRange{lo, lo + (rest < most ? rest : most)};
}

}  // namespace lbw
