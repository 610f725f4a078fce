// Which page holds a token: every index that a kernel takes from a page table goes through these, on the device and in
// the host's tests. Plain C++.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define LBW_LOOKUP __host__ __device__ __forceinline__
#else
#define LBW_LOOKUP inline
#endif

namespace lbw {

// The page that a table's entry names; -1: outside the cache of `pages`.
LBW_LOOKUP int page_of_entry(int32_t page, int pages) { return page >= 0 && page < pages ? page : -1; }

// The page of a sequence's token `row`, by its `width` table entries of 2^shift tokens each; -1: the table does not
// reach that far, or names a page outside the cache of `pages`.
LBW_LOOKUP int page_at(const int32_t* entries, int width, int shift, int pages, int64_t row) {
  if (row < 0 || (row >> shift) >= width) return -1;
  return page_of_entry(entries[row >> shift], pages);
}

// New tokens of a sequence that go into one page: t .. t + n - 1, rows row .. of the sequence, from row `in` of the page on.
struct PageRun {
  int t, n, in;
  int64_t row;
};
// Sequence b's tokens are start .. stop - 1 of a call's T, those of them that there are: `start` may lie before the first
// one and `stop` behind the last. Row r of its token t: len + t - start.
LBW_LOOKUP int first_token(int start) { return start > 0 ? start : 0; }
// Every page that new tokens go into has one owner. Told apart by pages: sequence b has the owners from first_owner on, 2^shift
// tokens each and as many as its tokens can touch pages, so that no sequence's lengths are wanted to find another's.
LBW_LOOKUP int64_t first_owner(int b, int start, int shift) { return (int64_t)(first_token(start) >> shift) + 2 * (int64_t)b; }
LBW_LOOKUP int64_t page_owners(int T, int B, int shift) { return (T >> shift) + 2 * (int64_t)B; }
// What owner first_owner + j looks after; false: no page.
LBW_LOOKUP bool owned_run(int start, int stop, int T, int len, int shift, int64_t j, PageRun& f) {
  const int mask = (1 << shift) - 1, first = first_token(start), end = stop < T ? stop : T;
  if (first >= end) return false;
  const int64_t row0 = (int64_t)len + ((int64_t)first - start);
  const int64_t row = j == 0 ? row0 : ((row0 >> shift) + j) * (mask + 1), t = first + (row - row0);
  if (t >= end) return false;
  f = PageRun{(int)t, 0, (int)(row & mask), row};
  f.n = end - f.t < mask + 1 - f.in ? end - f.t : mask + 1 - f.in;
  return true;
}
// Told apart by tokens: the first of a page's new ones owns it. `t` is the sequence's, at `row`; false: another one owns
// its page.
LBW_LOOKUP bool opened_run(int t, int64_t row, int start, int stop, int T, int shift, PageRun& f) {
  const int mask = (1 << shift) - 1, end = stop < T ? stop : T;
  f = PageRun{t, 0, (int)(row & mask), row};
  if (f.in != 0 && t != first_token(start)) return false;
  f.n = end - t < mask + 1 - f.in ? end - t : mask + 1 - f.in;
  return true;
}

// Half a tile of keys: 16 consecutive tokens of one page. `keys` of them are the sequence's; with BAD_PAGE added, their
// page is outside the cache (and `page` is 0, so that what is fetched all the same lies inside it).
constexpr int HALF_KEYS = 16;
constexpr int BAD_PAGE = 32;
struct Half {
  int page, keys;
};
// The half from place `pos` on (a multiple of 16) of a list of `span` places: the sequence's tokens in order, or (sel)
// those of the table entries that sel names, 2^shift places each. `len`: the sequence's keys.
LBW_LOOKUP Half half_at(const int32_t* sel, int64_t span, const int32_t* entries, int width, int shift, int pages,
                        int64_t len, int64_t pos) {
  // (the entry is read whatever the length, so that both can be on their way at once)
  int64_t row = pos;
  if (sel != nullptr) {
    if (pos >= span) return Half{0, 0};
    const int64_t entry = sel[pos >> shift];
    row = entry < 0 ? len : (entry << shift) + (pos & ((1 << shift) - 1));
  }
  const int page = page_at(entries, width, shift, pages, row);
  const int64_t left = (sel != nullptr || pos < span ? len - row : 0);
  if (left <= 0) return Half{0, 0};
  const int keys = left < HALF_KEYS ? (int)left : HALF_KEYS;
  return page >= 0 ? Half{page, keys} : Half{0, keys + BAD_PAGE};
}

}  // namespace lbw
