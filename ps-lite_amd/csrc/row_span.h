// The host's checks of where the rows of a call lie. (No GPU code: the host's tests compile it.)
#ifndef PSKV_ROW_SPAN_H_
#define PSKV_ROW_SPAN_H_
#include <stdint.h>

namespace pskv {

// n rows of k elements of `size` bytes, `stride` elements from one to the next.
struct RowSpan {
  const void* at;
  uint64_t n, k, stride, size;
  uint64_t begin() const { return reinterpret_cast<uintptr_t>(at); }
  uint64_t end() const { return begin() + ((n - 1) * stride + k) * size; }
};

// Whether two sets of rows share a byte. Rows that lie between each other's (columns of one matrix) do not.
inline bool rows_overlap(const RowSpan& a, const RowSpan& b) {
  if (!a.n || !b.n || !a.k || !b.k || a.end() <= b.begin() || b.end() <= a.begin()) return false;
  const uint64_t sa = a.stride * a.size, sb = b.stride * b.size;
  if (a.n == 1 && b.n == 1) return true;
  const uint64_t s = a.n == 1 ? sb : sa;
  if ((a.n > 1 && b.n > 1 && sa != sb) || s == 0) return true;
  // one step for both: where b's rows begin within a's step
  const uint64_t in = (b.begin() % s + s - a.begin() % s) % s;
  return in < a.k * a.size || in + b.k * b.size > s;
}

// A stretch of memory as one row (of nothing, if there is none).
inline RowSpan stretch(const void* at, uint64_t bytes) { return {at, 1, at ? bytes : 0, 0, 1}; }

// Whether two stretches of memory share a byte.
inline bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  return rows_overlap(stretch(a, a_bytes), stretch(b, b_bytes));
}

// A dimension: n of what the narrower ones make, `stride` bytes from one to the next.
struct Nest {
  uint64_t n, stride;
};

// Whether the bytes [first, behind) share one with a tensor: `row` bytes side by side, in `depth` dimensions that are sorted, the widest
// stride first, at `at`. (Dimensions that lie between each other are taken for what they reach together.)
inline bool touches(uint64_t first, uint64_t behind, uint64_t at, const Nest* dim, int depth, uint64_t row) {
  if (depth == 0) return row && first < behind && first < at + row && at < behind;
  uint64_t reach = row;
  for (int d = 1; d < depth; ++d) reach += (dim[d].n - 1) * dim[d].stride;
  const uint64_t s = dim[0].stride;
  if (dim[0].n < 2 || s == 0) return touches(first, behind, at, dim + 1, depth - 1, row);
  // the first and the last that begin before the end and end behind the beginning
  if (behind <= at) return false;
  const uint64_t low = first >= at + reach ? (first - at - reach) / s + 1 : 0, most = (behind - at - 1) / s;
  const uint64_t high = most < dim[0].n - 1 ? most : dim[0].n - 1;
  if (low > high) return false;
  if (high - low >= 2 || reach > s) return true;  // (one between them is covered whole)
  return touches(first, behind, at + low * s, dim + 1, depth - 1, row) ||
         (low != high && touches(first, behind, at + high * s, dim + 1, depth - 1, row));
}

// How many lanes serve a row of `vectors` vectors: a power of two, at most `most`.
inline unsigned lanes_for(uint64_t vectors, unsigned most) {
  unsigned lanes = 1;
  while (lanes < most && lanes < vectors) lanes <<= 1;
  return lanes;
}

}  // namespace pskv
#endif  // PSKV_ROW_SPAN_H_
