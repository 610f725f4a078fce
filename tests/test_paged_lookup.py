"""The one place where a kernel takes a page from a table (csrc/page_lookup.h), compiled for the host: whatever tables
and lists hold, it names pages inside the cache and tokens inside the page."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lingbot-world-v2_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "page_lookup.h"
using namespace lbw;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
  std::mt19937_64 g(1);
  auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(g); };
  const int32_t odd[] = {-1, -2147483647 - 1, 2147483647, 1 << 30, -7};
  for (int round = 0; round < 20000; ++round) {
    const int shift = (int)pick(4, 10), width = (int)pick(0, 9), pages = (int)pick(1, 12);
    std::vector<int32_t> entries(width), sel(pick(0, 6));   // (exactly as long as they may be read)
    for (auto& e : entries) e = pick(0, 3) ? (int32_t)pick(0, pages - 1) : (pick(0, 1) ? odd[pick(0, 4)] : pages);
    for (auto& e : sel) e = pick(0, 3) ? (int32_t)pick(0, width + 2) : odd[pick(0, 4)];
    const int64_t cap = (int64_t)width << shift, len = pick(0, cap);
    for (int64_t row : {(int64_t)-1, (int64_t)0, cap - 1, cap, pick(0, cap), (int64_t)1 << 40, -((int64_t)1 << 40)}) {
      const int p = page_at(entries.data(), width, shift, pages, row);
      CHECK(p >= -1 && p < pages);
      if (row < 0 || row >= cap) CHECK(p == -1);
      else CHECK(p == -1 ? entries[row >> shift] < 0 || entries[row >> shift] >= pages : p == entries[row >> shift]);
    }
    const bool list = pick(0, 1);
    const int64_t span = list ? (int64_t)sel.size() << shift : len;
    int64_t keys = 0;
    for (int64_t pos = 0; pos < span + 64; pos += HALF_KEYS) {
      const Half h = half_at(list ? sel.data() : nullptr, span, entries.data(), width, shift, pages, len, pos);
      CHECK(h.page >= 0 && h.page < pages);
      const int n = h.keys & (BAD_PAGE - 1);
      CHECK(h.keys >= 0 && h.keys < 2 * BAD_PAGE && n <= HALF_KEYS && (h.keys < BAD_PAGE || n > 0));
      // 16 tokens from a multiple of 16 on never leave their page
      CHECK((pos & ((1 << shift) - 1)) + HALF_KEYS <= 1 << shift);
      if (!list) keys += n;
      if (!list && h.keys < BAD_PAGE && n) CHECK(h.page == entries[pos >> shift]);
    }
    if (!list) CHECK(keys == len);
  }
  std::puts("ok");
  return 0;
}
"""


def test_lookups_stay_inside(tmp_path):
    src, exe = tmp_path / "lookup.cpp", tmp_path / "lookup"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr[-2000:]
