// Where the positions of sequences in pages lie (AhPages), for host and device.
#pragma once
#include <stdint.h>
#include "../../include/alpha_hip.h"

#if defined(__HIPCC__)
#define AH_BOTH __host__ __device__ __forceinline__
#else
#define AH_BOTH inline
#endif

namespace ah {

// Whole quotients by a number below 2^31 that is the same for a launch, of numerators below 2^31: with 2^(shift - 1) < divisor <= 2^shift and
// magic = ceil(2^(31 + shift) / divisor) < 2^32 (`shift` here has the 31 in it) the product n * magic is n * 2^(31 + shift) / divisor and less than 2^(31 + shift) / divisor more.
struct Quotient {
  uint32_t divisor, magic;
  int32_t  shift;
};
inline Quotient quotient_by(uint32_t divisor) {
  Quotient q{divisor, 0u, 31};
  while ((uint64_t(1) << (q.shift - 31)) < divisor) q.shift++;
  q.magic = (uint32_t)(((uint64_t(1) << q.shift) + divisor - 1) / divisor);
  return q;
}
AH_BOTH uint32_t quotient(uint32_t n, const Quotient &q) { return (uint32_t)(((uint64_t)n * q.magic) >> q.shift); }

constexpr int32_t MOST_POSITIONS = 0x7fff0000;      // so that a tile behind a position is still a position

struct PagedCache {
  const int32_t *table, *starts, *lens;
  int64_t  pages, page_stride, row_stride, head_stride;
  uint32_t page_pieces, row_pieces;      // strides of a page and of a row in 16 bytes
  Quotient page_rows;
  int32_t  seqs, table_pages;
  int32_t  rows;              // of the arrays of new tokens
  int32_t  capacity;          // positions that the table can name, at most MOST_POSITIONS
};

// Elements from the start of a page array to (position, head 0), from the page that the table names for it; negative: no such place.
AH_BOTH int64_t page_place(const PagedCache &c, int32_t page, uint32_t row) {
  return page >= 0 && page < c.pages ? page * c.page_stride + (int64_t)row * c.row_stride : -1;
}
AH_BOTH int64_t position_place(const PagedCache &c, int32_t seq, int32_t position) {
  if (position < 0 || position >= c.capacity) return -1;
  const uint32_t entry = quotient((uint32_t)position, c.page_rows);
  return page_place(c, c.table[(int64_t)seq * c.table_pages + entry], (uint32_t)position - entry * c.page_rows.divisor);
}
// What starts and lens say of a sequence: its first new row, how many, and its positions (those that the table cannot name among them)
struct Sequence { int32_t first, count, len; };
AH_BOTH Sequence sequence_of(int32_t start, int32_t next, int32_t len, int32_t rows) {
  Sequence s;
  s.first = start < 0 ? 0 : start > rows ? rows : start;
  const int32_t end = next < s.first ? s.first : next > rows ? rows : next;
  s.count = end - s.first;
  s.len = len < 0 ? 0 : len;
  return s;
}

// The host's half: the arguments that AhPages has, checked (paged.hip).
int32_t paged_cache(const char *who, const AhPages *p, int32_t rows, PagedCache *out);

}  // namespace ah
