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

// How many lanes serve a row of `vectors` vectors: a power of two, at most `most`.
inline unsigned lanes_for(uint64_t vectors, unsigned most) {
  unsigned lanes = 1;
  while (lanes < most && lanes < vectors) lanes <<= 1;
  return lanes;
}

}  // namespace pskv
#endif  // PSKV_ROW_SPAN_H_
