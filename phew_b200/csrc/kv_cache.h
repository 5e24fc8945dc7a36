// Index arithmetic of the paged, quantised key/value cache, shared by its
// kernels and plain C++ (the CPU tests compile this file with the host
// compiler, so nothing here needs CUDA).
//
// A cache side (keys or values) is [pages][kv_heads][page_size] token rows of
// head_dim codes.  Position `pos` of sequence b lies in page
// table[b][pos / page_size] at row pos % page_size, or in page b when there is
// no table.  Row numbers are 32-bit (the host refuses more than 2^32 - 2
// rows, which no 180 GB card holds); byte offsets are 64-bit.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define PHEW_HD __host__ __device__ __forceinline__
#else
#define PHEW_HD inline
#endif

namespace phew {
namespace kv {

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(m, n) + n) >> s
// (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994).
struct FastDiv {
  uint32_t d, m, s;
};

inline FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.s) < d) ++f.s;
  f.m = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.s) - d)) / d + 1);
  return f;
}

PHEW_HD uint32_t div_by(const FastDiv& f, uint32_t n) {
  const uint32_t hi = static_cast<uint32_t>((static_cast<uint64_t>(f.m) * n) >> 32);
  return (hi + n) >> f.s;
}

constexpr uint32_t kNoRow = 0xffffffffu;

// Where the pages of a batch lie.
struct PageMap {
  const int32_t* table;  // [batch][columns] page numbers, rows table_stride apart; null: page b
  int64_t table_stride;
  int32_t columns;  // pages a sequence can have (1 without a table)
  int32_t pages;    // pages in the cache
  int32_t kv_heads;
  int32_t page_size;
  FastDiv by_page;
};

// Tokens a sequence can have.
PHEW_HD int64_t capacity(const PageMap& m) { return static_cast<int64_t>(m.columns) * m.page_size; }

// Page number for column `col` of sequence b as the table gives it.
PHEW_HD int32_t page_at(const PageMap& m, int32_t b, int32_t col) {
  return m.table ? m.table[b * m.table_stride + col] : b;
}

PHEW_HD bool page_ok(const PageMap& m, int32_t page) { return page >= 0 && page < m.pages; }

// Row of token row `r` of a good page for head h.
PHEW_HD uint32_t row_at(const PageMap& m, int32_t page, int32_t h, int32_t r) {
  return (static_cast<uint32_t>(page) * static_cast<uint32_t>(m.kv_heads) + static_cast<uint32_t>(h)) *
             static_cast<uint32_t>(m.page_size) +
         static_cast<uint32_t>(r);
}

// Row of position `pos` of sequence b, head h; kNoRow when the position lies
// outside the sequence's pages or the table names no page of the cache.
PHEW_HD uint32_t row_of(const PageMap& m, int32_t b, int32_t h, int64_t pos) {
  if (pos < 0 || pos >= capacity(m)) return kNoRow;
  const int32_t col = static_cast<int32_t>(div_by(m.by_page, static_cast<uint32_t>(pos)));
  const int32_t page = page_at(m, b, col);
  if (!page_ok(m, page)) return kNoRow;
  return row_at(m, page, h, static_cast<int32_t>(pos) - col * m.page_size);
}

// A sequence's token count as the kernels use it: within [0, limit].
PHEW_HD int32_t clamp_count(int32_t n, int64_t limit) {
  if (n < 0) return 0;
  return n > limit ? static_cast<int32_t>(limit) : n;
}

// Keys [0, end) that query token `tok` of a sequence sees: with `causal` the
// last of its `count` query tokens sits at the sequence's last token.
PHEW_HD int32_t seen_end(int32_t length, int32_t count, int32_t tok, bool causal) {
  if (tok >= count) return 0;
  if (!causal) return length;
  const int32_t end = length - count + tok + 1;
  return end < 0 ? 0 : end;
}

}  // namespace kv
}  // namespace phew
