// The buckets of the relative position bias: which of a table's rows a key position gets from a query position.
//     rel = key - query;  two-sided: m = buckets / 2, d = |rel|, rows m.. where rel > 0;  one-sided: m = buckets, d = max(-rel, 0)
//     d < exact = m / 2: row d;  else row exact + floor((m - exact) log(d / exact) / log(max / exact)), at most m - 1
// A float's logarithm decides wrongly where its result is a whole number, and that is where the borders of common settings lie
// (exact 8, max 128: d = 16, 32, 64). So the borders are found as whole numbers: row exact + c begins at the least d with
//     d^(m - exact) >= exact^(m - exact - c) max^c.
// (No GPU code in here but bucket_of: the host's tests compile it.)
#ifndef PSKV_RELBIAS_H_
#define PSKV_RELBIAS_H_
#include <math.h>
#include <stdint.h>

#include <vector>

#ifdef __HIP__
#define PSKV_BOTH __host__ __device__
#else
#define PSKV_BOTH
#endif

namespace pskv {

constexpr unsigned kMostBuckets = 256;  // PSKV_RELBIAS_MAX_BUCKETS
constexpr uint64_t kMostDistance = 1ull << 30;

// Passed to the kernels by value.
struct Buckets {
  unsigned side;    // m
  unsigned exact;
  unsigned steps;   // borders in use
  unsigned two_sided;
  float log_exact, per_log;  // log2(exact), buckets per doubling of the distance
  uint32_t border[kMostBuckets / 2 + 1];  // 0, the least distances of the buckets that widen, the largest number
};

// Relative positions beyond the largest distance, and tiles of them, have one bucket: positions are kept to 32 bits.
PSKV_BOTH inline int32_t nearer(int64_t rel) {
  const int64_t most = (int64_t)kMostDistance + 65536;
  return rel > most ? (int32_t)most : rel < -most ? (int32_t)-most : (int32_t)rel;
}

// The same of rel0 - own + step: rel0 up to 2^61 and step up to 2^32 either way, `own` (a sequence's position) any number. From 2^62 on it
// alone decides on which side and that it is far, so its upper word may be brought nearer (two instructions of the scalar unit, which does not
// compare 64 bits).
PSKV_BOTH inline int32_t nearer(int64_t rel0, int64_t own, int64_t step) {
  const int32_t most = 1 << 30, upper = (int32_t)(own >> 32);
  const int32_t near = upper > most ? most : upper < -most ? -most : upper;
  return nearer(rel0 - (int64_t)((uint64_t)(uint32_t)near << 32 | (uint32_t)own) + step);
}

// The row of a relative position. The logarithm in float tells where to look: its error, some 1e-6, times at most 11,400 buckets per
// doubling is far below one, so the bucket is the one that it says or a neighbour, and the borders decide. `border` is b.border
// with 0 in front and the largest number behind, where it can be read fastest.
PSKV_BOTH inline unsigned bucket_of(const Buckets& b, const uint32_t* border, int32_t rel) {
  const bool ahead = b.two_sided && rel > 0;
  const uint32_t d = ahead ? (uint32_t)rel : rel < 0 ? 0 - (uint32_t)rel : 0;
#ifdef __HIP_DEVICE_COMPILE__
  const float log = __builtin_amdgcn_logf((float)d);
#else
  const float log = log2f((float)d);
#endif
  float guess = (log - b.log_exact) * b.per_log;
  guess = guess > 0.0f ? guess : 0.0f;
  const unsigned c = guess < (float)b.steps ? (unsigned)guess : b.steps;
  const unsigned row = d < b.exact ? d : b.exact + c + (d >= border[c + 1] ? 1 : 0) - (d < border[c] ? 1 : 0);
  return ahead ? b.side + row : row;
}

// A whole number of any length, for the few comparisons that a double cannot decide.
struct Whole {
  std::vector<uint32_t> digit{1};
  void times(uint32_t x) {
    uint64_t carry = 0;
    for (uint32_t& d : digit) {
      carry += (uint64_t)d * x;
      d = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) digit.push_back((uint32_t)carry);
  }
  bool operator>=(const Whole& o) const {
    if (digit.size() != o.digit.size()) return digit.size() > o.digit.size();
    for (size_t i = digit.size(); i-- > 0;)
      if (digit[i] != o.digit[i]) return digit[i] > o.digit[i];
    return true;
  }
};

// d^n >= exact^(n - c) max^c
inline bool at_border(uint64_t d, unsigned n, unsigned c, uint64_t exact, uint64_t max) {
  unsigned x = n, y = c;  // the greatest common divisor of n and c goes
  while (y) {
    const unsigned r = x % y;
    x = y;
    y = r;
  }
  n /= x;
  c /= x;
  Whole left, right;
  for (unsigned i = 0; i < n; ++i) {
    left.times((uint32_t)d);
    right.times((uint32_t)(i < c ? max : exact));
  }
  return left >= right;
}

// false: not a setting that makes sense. (May throw std::bad_alloc.)
inline bool make_buckets(Buckets* b, uint64_t buckets, uint64_t max_distance, bool two_sided) {
  if (buckets > kMostBuckets || max_distance > kMostDistance) return false;
  b->two_sided = two_sided ? 1 : 0;
  b->side = (unsigned)(two_sided ? buckets / 2 : buckets);
  if (b->side < 2) return false;
  b->exact = b->side / 2;
  if (max_distance <= b->exact) return false;
  const unsigned n = b->side - b->exact;
  b->steps = n - 1;
  b->log_exact = (float)log2((double)b->exact);
  b->per_log = (float)(n / log2((double)max_distance / b->exact));
  const double grow = log((double)max_distance / b->exact) / n;
  for (unsigned c = 1; c < n; ++c) {
    const double r = b->exact * exp(grow * c);
    // r is right to some 1e-14 of itself: where no whole number is that near, the border is the next one
    const double near = r * 1e-12;
    uint64_t d = (uint64_t)ceil(r - near);
    const uint64_t most = (uint64_t)floor(r + near);
    while (d <= most && !at_border(d, n, c, b->exact, max_distance)) ++d;
    b->border[c] = (uint32_t)d;
  }
  b->border[0] = 0;
  b->border[n] = ~0u;
  return true;
}

}  // namespace pskv
#endif  // PSKV_RELBIAS_H_
