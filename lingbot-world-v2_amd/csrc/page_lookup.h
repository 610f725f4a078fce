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
