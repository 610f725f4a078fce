"""The search for the last chosen page's score (csrc/score_range.h), compiled for the host: bins hold what was counted into
them, every search ends, and the border is the one that sorting finds -- with infinite, negative, tiny and equal scores."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lingbot-world-v2_amd", "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>
#include <random>
#include <vector>
#include "score_range.h"
using namespace lbw;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return false; } } while (0)

uint64_t image(double x) {
  x += 0.0;
  uint64_t u;
  std::memcpy(&u, &x, 8);
  return (u >> 63) ? ~u : u | (1ull << 63);
}

// The kernel's search, one thread for all: the need-th highest of `scores` (0: none), by as many as `most` at the end.
bool search(const std::vector<uint64_t>& scores, uint32_t need, uint32_t most) {
  std::vector<uint64_t> sorted;
  for (uint64_t u : scores)
    if (u != 0) sorted.push_back(u);
  std::sort(sorted.rbegin(), sorted.rend());
  CHECK(need >= 1 && need <= sorted.size());
  const uint64_t want = sorted[need - 1];
  ScoreRange r{sorted.back(), sorted[0]};
  for (int round = 0;; ++round) {
    CHECK(round < 8);                       // 64 bits, ten less a round: 54, 44, .., 4, one score
    CHECK(r.lo <= want && want <= r.hi);
    if (r.lo == r.hi) return true;
    const int shift = bin_shift(r);
    std::vector<uint32_t> hist(SCORE_BINS, 0);
    for (uint64_t u : scores)
      if (in_range(r, u)) {
        const int bin = bin_of(r, shift, u);
        CHECK(bin >= 0 && bin < SCORE_BINS);
        ++hist[bin];
      }
    int bin = SCORE_BINS;
    uint32_t upto = 0;
    while (bin-- > 0 && upto + hist[bin] < need) upto += hist[bin];
    CHECK(bin >= 0);
    need -= upto;
    r = bin_range(r, shift, bin);
    CHECK(r.lo <= r.hi);
    uint32_t there = 0;
    for (uint64_t u : scores) there += in_range(r, u);
    CHECK(there == hist[bin]);              // what is collected fits where it was counted to fit
    if (need == hist[bin]) {
      CHECK(*std::min_element(sorted.begin(), sorted.begin() + (std::upper_bound(sorted.begin(), sorted.end(), want,
                              std::greater<uint64_t>()) - sorted.begin())) == want);
      for (uint64_t u : scores) CHECK(u == 0 || (u > r.lo - 1) == (u >= want));
      return true;
    }
    if (there <= most) return true;
  }
}

int main() {
  const double inf = std::numeric_limits<double>::infinity();
  std::mt19937_64 g(1);
  auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(g); };
  auto real = [&](double lo, double hi) { return std::uniform_real_distribution<double>(lo, hi)(g); };
  // finite scores from `low` up, more infinite ones than are wanted
  for (double low : {-1e300, -1e30, -100.0, -50.0, -20.0, -10.0, -5.0, -3.0, -1.0, -1e-300, 0.0, 1e-300, 0.3, 0.5, 0.7, 0.99,
                     1.0, 1.5, 2.0, 1e30, 1e300, -inf})
    for (int finite : {1, 91, 200, 400})
      for (int infinite : {2, 9, 300, 600})
        for (uint32_t need : {1u, 4u, (uint32_t)infinite - 1, (uint32_t)infinite})
          for (uint32_t most : {1u, 256u, 512u}) {
            std::vector<uint64_t> s(finite, image(low));
            for (int i = 1; i < finite; ++i) s[i] = image(std::isinf(low) || std::abs(low) > 1e20 ? low : low + 0.01 * i);
            s.insert(s.end(), infinite, image(inf));
            s.push_back(0);
            if (need <= (uint32_t)infinite && !search(s, need, most)) {
              std::printf("low %g, %d finite, %d infinite, need %u, most %u\n", low, finite, infinite, need, most);
              return 1;
            }
          }
  // any bits at all, few and many of a kind
  for (int round = 0; round < 20000; ++round) {
    std::vector<uint64_t> s(pick(1, 300));
    const int kind = (int)pick(0, 4);
    for (auto& u : s) {
      if (kind == 0) u = std::max<uint64_t>(1, std::min<uint64_t>(g(), image(inf)));
      else if (kind == 1) u = image(std::ldexp(real(-1, 1), (int)pick(-1000, 1000)));
      else if (kind == 2) u = image(real(-3, 3));
      else if (kind == 3) u = image((double)pick(-2, 2));
      else u = image(inf) - (uint64_t)pick(0, 5);
      if (pick(0, 9) == 0) u = image(pick(0, 1) ? inf : -inf);
    }
    if (!search(s, (uint32_t)pick(1, (int64_t)s.size()), (uint32_t)pick(1, 40))) return 1;
  }
  std::puts("ok");
  return 0;
}
"""


def test_the_border_is_found(tmp_path):
    src, exe = tmp_path / "border.cpp", tmp_path / "border"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr[-2000:]
