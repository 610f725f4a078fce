"""Who looks after the pages that new tokens go into (csrc/page_lookup.h), compiled for the host: told apart by pages or by
tokens, every token of a sequence is in one owner's run, at its row and inside one page -- wherever the starts lie."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lingbot-world-v2_amd", "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "page_lookup.h"
using namespace lbw;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return false; } } while (0)

struct Call {
  int T, shift;
  std::vector<int> starts, lens;
};

bool mark(const Call& c, int b, const PageRun& f, std::vector<int>& seen) {
  CHECK(f.n > 0 && f.t >= 0 && f.t + f.n <= c.T && f.t >= c.starts[b] && f.t + f.n <= c.starts[b + 1]);
  CHECK(f.row == (int64_t)c.lens[b] + ((int64_t)f.t - c.starts[b]));
  CHECK(f.in == (f.row & ((1 << c.shift) - 1)) && f.in + f.n <= 1 << c.shift);
  for (int t = f.t; t < f.t + f.n; ++t) ++seen[t];
  return true;
}

bool check(const Call& c) {
  const int B = (int)c.lens.size();
  std::vector<int> want(c.T, 0), pages(c.T, 0), tokens(c.T, 0);
  std::vector<int> of(c.T, -1);
  for (int b = 0; b < B; ++b)
    for (int64_t t = std::max(c.starts[b], 0); t < std::min(c.starts[b + 1], c.T); ++t) want[t] = 1, of[t] = b;
  const int64_t owners = page_owners(c.T, B, c.shift);
  for (int64_t slot = 0; slot < owners; ++slot) {
    int b = -1;
    for (int x = 0; x < B; ++x)
      if (first_owner(x, c.starts[x], c.shift) <= slot) b = x;
    PageRun f;
    if (b >= 0 && owned_run(c.starts[b], c.starts[b + 1], c.T, c.lens[b], c.shift,
                            slot - first_owner(b, c.starts[b], c.shift), f))
      CHECK(mark(c, b, f, pages));
  }
  CHECK(pages == want);
  for (int t = 0; t < c.T; ++t) {
    const int b = of[t];
    PageRun f;
    if (b >= 0 && opened_run(t, (int64_t)c.lens[b] + ((int64_t)t - c.starts[b]), c.starts[b], c.starts[b + 1], c.T, c.shift, f))
      CHECK(mark(c, b, f, tokens));
  }
  CHECK(tokens == want);
  return true;
}

int main() {
  for (int shift = 4; shift <= 10; ++shift)
    for (const Call& c : {Call{100, shift, {-5, 100}, {0}}, Call{100, shift, {-200, 100}, {3}}, Call{4, shift, {-2, 2}, {5}},
                          Call{40, shift, {-2147483647 - 1, -3, 7, 40}, {0, 9, 15}}, Call{30, shift, {7}, {}},
                          Call{50, shift, {0, 2147483647}, {2147483647 - 20}}, Call{50, shift, {-2147483647, 2147483647}, {-9}}})
      if (!check(c)) {
        std::printf("shift %d, T %d, first start %d\n", shift, c.T, c.starts[0]);
        return 1;
      }
  std::mt19937_64 g(1);
  auto pick = [&](int64_t lo, int64_t hi) { return (int)std::uniform_int_distribution<int64_t>(lo, hi)(g); };
  for (int round = 0; round < 30000; ++round) {
    Call c{pick(1, 300), pick(4, 7), {}, std::vector<int>(pick(0, 12))};
    for (auto& x : c.lens) x = pick(0, 9) ? pick(0, 200) : pick(-40, 0);
    c.starts.resize(c.lens.size() + 1);
    const int from = pick(0, 2) ? 0 : -pick(0, 300), to = pick(0, 2) ? c.T : c.T + pick(-c.T, 300);
    for (auto& x : c.starts) x = pick(std::min(from, to), std::max(from, to));
    std::sort(c.starts.begin(), c.starts.end());
    if (!check(c)) return 1;
  }
  std::puts("ok");
  return 0;
}
"""


def test_every_token_has_one_owner(tmp_path):
    src, exe = tmp_path / "owners.cpp", tmp_path / "owners"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr[-2000:]


@pytest.mark.parametrize("page", [16, 64, 128, 256, 1024])
@pytest.mark.parametrize("tokens", [1, 64, 65, 100, 255, 1000])
def test_tokens_of_no_sequence_are_no_launch(page, tokens):
    """A batch of none: every token belongs to nobody, so there is nothing to do (and no device is wanted)."""
    import ctypes

    from lbw_amd import _lib
    from test_paged_host import ADDR, _append
    for bounds in (ADDR, None):
        p = _append(tokens=tokens, batch=0, starts=ADDR, lens=None, **{"cache.page_size": page, "cache.bounds": bounds})
        assert _lib.load().lbw_paged_append(ctypes.byref(p), None) == 0
