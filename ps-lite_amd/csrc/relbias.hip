// The learned relative position bias and its gradient (gfx950):
//     out[b,h,i,j] = scores[b,h,i,j] + table[bucket(rel)][h],  rel = (k_first + j) - (q_first + q_at[b] + i)
//     dtable[u][h] = sum of grad[b,h,i,j] over the b, i, j whose bucket is u
// The bias depends on j - i alone. Both directions go by tiles of a wavefront whose lanes hand values to each other along the
// diagonals; the gradient's diagonals are summed into buckets once per tile.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>

#include "host_common.h"
#include "lanes.h"
#include "relbias.h"
#include "row_types.h"

namespace pskv {
namespace {

constexpr unsigned kBlock = 256;
constexpr unsigned kWaves = kBlock / 64;
constexpr unsigned kGroup = 8;           // rows that a wavefront asks for before it uses them
constexpr unsigned kMostRows = 128;      // of a wavefront
constexpr uint64_t kMostTiles = 1u << 31;

struct Shape {
  uint64_t B, H, Q, K;
  int64_t rel0;  // of row 0, column 0, before q_at
  uint64_t in[3], out[3];  // strides of batch, head and row
};

// How a call is cut up: a wavefront takes `rows` rows of `cols` columns, for `heads` heads and `batches` batches one after the other.
struct Cut {
  unsigned cols, rows, heads, batches;
  unsigned across, strips, parts, chunks;  // how many there are of columns, rows, heads, batches
  uint64_t tiles() const { return (uint64_t)across * strips * parts * chunks; }
};

// N neighbouring elements, as they are in memory and as numbers.
template <typename T, unsigned N>
struct Some {
  static constexpr int kWords = (int)(N * sizeof(T) / 4);
  uint32_t word[kWords];

  template <bool PAST>
  __device__ __forceinline__ void load(const T* p) {
    typedef uint32_t Quad __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int q = 0; q < kWords / 4; ++q) {
      const Quad v = __builtin_bit_cast(Quad, get<PAST>(p + q * Row<T>::kWide));
#pragma unroll
      for (int i = 0; i < 4; ++i) word[4 * q + i] = v[i];
    }
  }
  // n (up to N) of them, zeros behind them.
  __device__ __forceinline__ void few(const T* p, unsigned n) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = 0;
#pragma unroll
    for (unsigned i = 0; i < N; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4)
          word[i] = __builtin_bit_cast(uint32_t, p[i]);
        else
          word[i / 2] |= (uint32_t)__builtin_bit_cast(unsigned short, p[i]) << (i & 1 ? 16 : 0);
      }
  }
  // The elements from `off` (up to N) on, zeros behind them: what a lane at the end of a row needs that has loaded the last N.
  __device__ __forceinline__ void skip(unsigned off) {
    constexpr int kHalf = sizeof(T) == 2 ? 1 : 0;
    if (kHalf) {
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        word[i] = __builtin_amdgcn_alignbit(i + 1 < kWords ? word[i + 1] : 0u, word[i], off & 1 ? 16 : 0);
    }
#pragma unroll
    for (int step = 1; step <= kWords; step <<= 1) {
      const bool now = ((off >> kHalf) & (unsigned)step) != 0;
#pragma unroll
      for (int i = 0; i < kWords; ++i) word[i] = now ? (i + step < kWords ? word[i + step] : 0u) : word[i];
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (std::is_same<T, float>::value)
      return __builtin_bit_cast(float, word[i]);
    else if constexpr (std::is_same<T, __bf16>::value)
      return __builtin_bit_cast(float, i & 1 ? word[i / 2] & 0xffff0000u : word[i / 2] << 16);
    else
      return (float)__builtin_bit_cast(_Float16, (unsigned short)(i & 1 ? word[i / 2] >> 16 : word[i / 2]));
  }
};

// Rounds N numbers and stores the first n of them.
template <bool PAST, unsigned N, typename T>
__device__ __forceinline__ void store_some(T* p, const float (&y)[N], unsigned n) {
  constexpr unsigned kSome = Row<T>::kWide;
  T e[N];
#pragma unroll
  for (unsigned i = 0; i < N; ++i) e[i] = (T)y[i];
  if (n == N) {
#pragma unroll
    for (unsigned q = 0; q < N / kSome; ++q) {
      typename Row<T>::Vec v;
#pragma unroll
      for (unsigned i = 0; i < kSome; ++i) v[i] = e[q * kSome + i];
      put<PAST>(p + q * kSome, v);
    }
    return;
  }
  // four, two and one of them
  typedef T Two __attribute__((ext_vector_type(2), aligned(sizeof(T))));
  typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const unsigned done = N > 4 ? n & 4 : 0;
  if (done) *reinterpret_cast<Four*>(p) = Four{e[0], e[1], e[2], e[3]};
  const T a = done ? e[N - 4] : e[0], b = done ? e[N - 3] : e[1], c = done ? e[N - 2] : e[2];
  if (n & 2) *reinterpret_cast<Two*>(p + done) = Two{a, b};
  if (n & 1) p[done + (n & 2)] = n & 2 ? c : a;
}

// A lane's part of the rows of a tile: columns c to c + N - 1, or what there is of them.
template <unsigned N>
struct Span {
  uint64_t at;     // where it loads: at c, or the last N of the row
  unsigned off;    // how many of those come before c
  unsigned own;    // columns, 0 to N
  bool ends, few;  // the same for the wavefront: the row ends within its columns; it is shorter than a load
  __device__ __forceinline__ Span(uint64_t c0, unsigned lane, uint64_t K) {
    const uint64_t c = c0 + lane * N;
    ends = c0 + 64 * N > K;
    few = K < N;
    own = c >= K ? 0 : K - c < N ? (unsigned)(K - c) : N;
    at = few || own == N ? c : K - N;
    off = c - at < N ? (unsigned)(c - at) : N;
  }
  // kGroup rows, or the first n of them where not WHOLE. (All of them are asked for before any is touched.)
  template <bool WHOLE, bool PAST, typename T>
  __device__ __forceinline__ void load(Some<T, N> (&x)[kGroup], const T* row, uint64_t stride, unsigned n) const {
    if (few) {
#pragma unroll
      for (unsigned r = 0; r < kGroup; ++r)
        if (WHOLE || r < n) x[r].few(row + r * stride + at, own);
      return;
    }
#pragma unroll
    for (unsigned r = 0; r < kGroup; ++r)
      if (WHOLE || r < n) x[r].template load<PAST>(row + r * stride + at);
    if (ends) {
#pragma unroll
      for (unsigned r = 0; r < kGroup; ++r)
        if (WHOLE || r < n) x[r].skip(off);
    }
  }
};

// The tile of a wavefront.
struct Tile {
  uint64_t c0, r0;  // the first column and row
  unsigned head0, batch0, rows, heads, batches;
  __device__ __forceinline__ Tile(unsigned tile, const Cut& cut, const Shape& s) {
    c0 = (uint64_t)(tile % cut.across) * cut.cols;
    tile /= cut.across;
    r0 = (uint64_t)(tile % cut.strips) * cut.rows;
    tile /= cut.strips;
    head0 = tile % cut.parts * cut.heads;
    batch0 = tile / cut.parts * cut.batches;
    rows = s.Q - r0 < cut.rows ? (unsigned)(s.Q - r0) : cut.rows;
    heads = (unsigned)s.H - head0 < cut.heads ? (unsigned)s.H - head0 : cut.heads;
    batches = (unsigned)s.B - batch0 < cut.batches ? (unsigned)s.B - batch0 : cut.batches;
  }
};

// The borders in LDS, for the workgroup. (A barrier has to follow.)
__device__ __forceinline__ void fetch_borders(uint32_t* to, const Buckets& b) {
  for (unsigned c = threadIdx.x; c < b.steps + 2; c += kBlock) to[c] = b.border[c];
}

// The bias, eight rows to a wavefront, of 16 bytes of columns to a lane, of one head. A row's bias is that of the row
// above, moved one column to the right, so what eight rows need is the first row's and the eight columns to the left of it, which
// the lanes below have: one look-up for eight elements. Bound by memory: scores of 4 x 16 x 2048 x 2048 bf16 at 5.7 TB/s (189 us; 32
// rows to a wavefront 215: what is at work is spread over more memory; the table staged in LDS: no gain), the bias alone of
// 12 x 1023 x 1023 float32 in 11.6 us (8 columns to a lane in two halves: 17.9), rows that begin at odd elements no slower than
// others (16 x 2048 x 2047 float16 57 us).
template <typename T, bool SCORES, bool PAST>
__global__ __launch_bounds__(kBlock) void k_relbias(const float* __restrict__ table, const int64_t* __restrict__ q_at,
                                                     const T* scores, T* out, unsigned tiles, Cut cut, Shape s, Buckets b) {
  constexpr unsigned N = Row<T>::kWide;
  __shared__ uint32_t border[kMostBuckets / 2 + 1];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  fetch_borders(border, b);
  __syncthreads();
  for (unsigned tile = blockIdx.x * kWaves + wave; tile < tiles; tile += gridDim.x * kWaves) {
    const Tile t(tile, cut, s);
    const Span<N> span(t.c0, lane, s.K);
    const int32_t rel = nearer(s.rel0, q_at ? q_at[t.batch0] : 0, (int64_t)(t.c0 - t.r0));
    unsigned row[N];  // of the table
#pragma unroll
    for (unsigned k = 0; k < N; ++k) row[k] = bucket_of(b, border, rel + (int)(lane * N + k)) * (unsigned)s.H;
    // the eight columns to the left of the tile: lanes 0 to 7 have one each
    const unsigned left = bucket_of(b, border, rel - (int)kGroup + (int)(lane & (kGroup - 1))) * (unsigned)s.H;
    const uint64_t head = t.head0;
    const T* from = SCORES ? scores + t.batch0 * s.in[0] + head * s.in[1] + t.r0 * s.in[2] : nullptr;
    T* to = out + t.batch0 * s.out[0] + head * s.out[1] + t.r0 * s.out[2] + t.c0 + lane * N;
    auto group = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      Some<T, N> x[kGroup];
      if (SCORES) span.template load<WHOLE, PAST>(x, from, s.in[2], t.rows);
      float v[kGroup + N];  // v[kGroup + k]: of the first row's column k
      const float corner = table[left + head];
#pragma unroll
      for (unsigned k = 0; k < N; ++k) v[kGroup + k] = table[row[k] + head];
      // handed up from the lane below, N columns at a time
#pragma unroll
      for (int k = kGroup - 1; k >= 0; --k)
        v[k] = from_below(v[k + N], __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, corner), k)));
#pragma unroll
      for (unsigned r = 0; r < kGroup; ++r) {
        if (!WHOLE && r >= t.rows) continue;
        float y[N];
#pragma unroll
        for (unsigned k = 0; k < N; ++k) y[k] = SCORES ? x[r].at(k) + v[kGroup + k - r] : v[kGroup + k - r];
        store_some<PAST>(to + r * s.out[2], y, span.own);
      }
    };
    if (t.rows == kGroup)
      group(std::true_type());
    else
      group(std::false_type());
  }
}

// One query to a sequence: a wavefront takes the same columns of eight heads (or fewer), whose rows of the table are the same.
// 64 sequences x 16 heads x 4,096 keys bf16: 7.4 to 8.1 us (head by head 9.2): a start, a look-up, 17 MB.
template <typename T, bool SCORES>
__global__ __launch_bounds__(kBlock) void k_relbias_step(const float* __restrict__ table, const int64_t* __restrict__ q_at,
                                                          const T* scores, T* out, unsigned tiles, Cut cut, Shape s, Buckets b) {
  constexpr unsigned N = Row<T>::kWide;
  __shared__ uint32_t border[kMostBuckets / 2 + 1];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  fetch_borders(border, b);
  __syncthreads();
  for (unsigned tile = blockIdx.x * kWaves + wave; tile < tiles; tile += gridDim.x * kWaves) {
    const Tile t(tile, cut, s);
    const Span<N> span(t.c0, lane, s.K);
    auto heads = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      Some<T, N> x[kGroup];
      if (SCORES)
        span.template load<WHOLE, false>(x, scores + t.batch0 * s.in[0] + t.head0 * s.in[1], s.in[1], t.heads);
      const int32_t rel = nearer(s.rel0, q_at ? q_at[t.batch0] : 0, (int64_t)t.c0);
      unsigned row[N];
#pragma unroll
      for (unsigned k = 0; k < N; ++k) row[k] = bucket_of(b, border, rel + (int)(lane * N + k)) * (unsigned)s.H + t.head0;
      T* to = out + t.batch0 * s.out[0] + t.head0 * s.out[1] + t.c0 + lane * N;
#pragma unroll
      for (unsigned h = 0; h < kGroup; ++h) {
        if (!WHOLE && h >= t.heads) continue;
        float y[N];
#pragma unroll
        for (unsigned k = 0; k < N; ++k) y[k] = SCORES ? x[h].at(k) + table[row[k] + h] : table[row[k] + h];
        store_some<false>(to + h * s.out[1], y, span.own);
      }
    };
    if (t.heads == kGroup)
      heads(std::true_type());
    else
      heads(std::false_type());
  }
}

// --- narrow matrices ---------------------------------------------------------------------------------------------

// A wavefront whose lanes are one row's columns has little to do where there are few of them. There a workgroup takes a plane: as
// many whole rows as kPlane elements hold, its lanes going through them cell by cell, 2 or 4 bytes at a time. That costs by the
// cell: 16.8 M of them in 1,024 matrices take the bias of scores 27 to 30 us, alone 24, the gradient in bf16 28 to 30 and in
// float32 17, and 45 and 36 where each sequence has its own position. By columns they take (bf16; 1, 16, 49 of them)
//     scores 2306, 160, 66   alone 1363, 90, 36   gradient 1170, 64, 49   own positions 1927, 113, 58
// and less than by planes from where these rules end (bf16, float32; planes behind the arrow):
//     scores in bf16, 112 columns: 29.6 -> 26.2; 120: 27.1 -> 28.5   in float32, 80: 29.4 -> 28.8; 96: 27.4 -> 28.5
//     alone, 63: 34 -> 24, 29 -> 24; 64, whose rows begin at whole lines: 27.8 -> 24.9, 22.1 -> 24.5; 80: 23.5 -> 24.8, 19.0 -> 23.9
//     gradient, 120: 30.8 -> 28.2, 35 -> 17 (80, whose rows do so in bf16: 26.3 -> 28.7, 31.7 -> 16.8); 128: 19.6 -> 28.3, 22.5 -> 16.7
//     own positions, 63: 56 -> 46, 58 -> 36; 64: 31 -> 47, 35 -> 36
constexpr unsigned kPlane = 2048;
constexpr unsigned kEach = kPlane / kBlock;  // cells of a lane
uint64_t plane_rows(size_t Q, size_t K) { return kPlane / (K | 1) < Q ? kPlane / (K | 1) : Q; }
bool tall(size_t Q, size_t K) { return K <= kPlane / 2 && Q / ((Q + plane_rows(Q, K) - 1) / plane_rows(Q, K)) >= 28; }
// Where each sequence has its own position, a plane is looked up or summed into buckets for one of them: what that takes, as long
// as some 20 rows by columns, has to be worth it (8,192 or 4,096 sequences, 16 heads; scores in bf16, float32, gradient in bf16, float32):
//     8 x 8:   159 -> 334, 112 -> 351, 239 -> 352, 266 -> 346     16 x 16: 312 -> 369, 215 -> 368, 338 -> 366, 368 -> 355
//     30 x 30: 323 -> 209, 270 -> 250, 302 -> 222, 339 -> 191     50 x 5:  655 -> 187, 371 -> 187, 656 -> 176, 511 -> 174
// (49 x 49, two planes of 24 rows, 2,048 sequences: 314 -> 283, 239 -> 309, 246 -> 297, 257 -> 244).
bool by_planes(size_t Q, size_t K, size_t size, bool scores, bool own_positions) {
  return Q > 1 && K <= (!scores ? 63 : size == 2 ? 112 : 80) && (!own_positions || tall(Q, K));
}
bool sums_by_planes(size_t Q, size_t K, bool own_positions) { return own_positions ? K <= 63 && tall(Q, K) : K <= 127; }

struct Plane {
  unsigned row[kEach], col[kEach];  // (of cells that are not there: the first)
  unsigned passes, cells;           // the same for the workgroup
  __device__ __forceinline__ Plane(unsigned rows, unsigned K) {
    cells = rows * K;
    passes = (cells + kBlock - 1) / kBlock;
    const unsigned down = kBlock / K, along = kBlock - down * K;
    unsigned r = threadIdx.x / K, k = threadIdx.x - r * K;
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) {
      row[i] = has(i) ? r : 0;
      col[i] = has(i) ? k : 0;
      r += down, k += along;
      if (k >= K) k -= K, ++r;
    }
  }
  __device__ __forceinline__ bool has(unsigned i) const { return threadIdx.x + i * kBlock < cells; }
};

// The bias of a plane's diagonals, looked up once for all its batches.
template <typename T, bool SCORES>
__global__ __launch_bounds__(kBlock) void k_relbias_narrow(const float* __restrict__ table, const int64_t* __restrict__ q_at,
                                                            const T* scores, T* out, unsigned tiles, Cut cut, Shape s, Buckets b) {
  __shared__ uint32_t border[kMostBuckets / 2 + 1];
  __shared__ float bias[kPlane];  // (rows + K - 1 <= rows K)
  fetch_borders(border, b);
  const unsigned K = (unsigned)s.K;
  for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const Tile t(tile, cut, s);
    const Plane c(t.rows, K);
    const int32_t rel = nearer(s.rel0, q_at ? q_at[t.batch0] : 0, (int64_t)(0 - t.r0 - (t.rows - 1)));
    __syncthreads();
    for (unsigned x = threadIdx.x; x < t.rows + K - 1; x += kBlock)
      bias[x] = table[bucket_of(b, border, rel + (int)x) * (unsigned)s.H + t.head0];
    __syncthreads();
    const T* from = SCORES ? scores + t.batch0 * s.in[0] + t.head0 * s.in[1] + t.r0 * s.in[2] : nullptr;
    T* to = out + t.batch0 * s.out[0] + t.head0 * s.out[1] + t.r0 * s.out[2];
    float v[kEach];
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) v[i] = c.has(i) ? bias[t.rows - 1 + c.col[i] - c.row[i]] : 0.0f;
    for (unsigned n = 0; n < t.batches; ++n) {
      T x[kEach];
      if (SCORES) {
#pragma unroll
        for (unsigned i = 0; i < kEach; ++i)
          if (i < c.passes) x[i] = from[n * s.in[0] + c.row[i] * s.in[2] + c.col[i]];
      }
#pragma unroll
      for (unsigned i = 0; i < kEach; ++i)
        if (c.has(i)) to[n * s.out[0] + c.row[i] * s.out[2] + c.col[i]] = (T)(SCORES ? (float)x[i] + v[i] : v[i]);
    }
  }
}

// --- the gradient ------------------------------------------------------------------------------------------------

// Adds diagonals x of `from`, `from` + `step`, ... below `count`, 64 neighbours at a time, to a wavefront's sums of their buckets;
// `rel` is diagonal 0's relative position. Far from the main diagonal 64 of them have one bucket: those are added up lane by lane
// until another one comes.
template <typename F>
__device__ __forceinline__ void add_buckets(float* sums, const Buckets& b, const uint32_t* border, int32_t rel, unsigned from,
                                            unsigned step, unsigned count, F value) {
  const unsigned lane = threadIdx.x & 63;
  float run = 0.0f;
  unsigned now = kMostBuckets;
  auto finish = [&] {
    if (now == kMostBuckets) return;
    run = sum_along(run, 0);
    if (lane == 63) sums[now] += run;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    run = 0.0f;
    now = kMostBuckets;
  };
  for (unsigned x0 = from; x0 < count; x0 += step) {
    const unsigned x = x0 + lane;
    float sum = x < count ? value(x) : 0.0f;
    const unsigned u = bucket_of(b, border, rel + (int)x), first = __builtin_amdgcn_readfirstlane(u);
    if (__all(u == first)) {
      if (first != now) finish();
      now = first;
      run += sum;
      continue;
    }
    finish();
    // lanes of one bucket are neighbours: a sum over each stretch of them, left at its last lane
    const unsigned below = dpp<0x138 /* wave_shr:1 */, 0xf>(u), above = dpp<0x130 /* wave_shl:1 */, 0xf>(u);
    sum = sum_along(sum, lane == 0 || below != u ? 1 : 0);
    if (lane == 63 || above != u) sums[u] += sum;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  finish();
}

// The wavefronts' sums of a workgroup. (Behind a barrier.)
__device__ __forceinline__ void put_sums(const float (&sums)[kWaves][kMostBuckets], float* to, uint64_t by_bucket, unsigned buckets) {
  for (unsigned u = threadIdx.x; u < buckets; u += kBlock) {
    float sum = sums[0][u];
#pragma unroll
    for (unsigned w = 1; w < kWaves; ++w) sum += sums[w][u];
    to[u * by_bucket] = sum;
  }
}

constexpr unsigned kWide = 8;           // neighbouring columns of a lane
constexpr unsigned kCols = 64 * kWide;  // of a wavefront

// The same the other way round: rows are summed over the batch, then along the diagonals, which move up one lane every
// eight rows; those that leave lane 63 and those that are there in the end are summed by bucket, 64 neighbouring diagonals
// at a time. Every sum has one order. `to`: [head][bucket][workgroup of the head], or the gradient itself where a head has one
// workgroup. 8 x 16 x 1024 x 1024 bf16: 45 us, 6.0 TB/s, and 5 for
// k_relbias_join (a lane to a diagonal, element by element: 460).
template <typename T, bool PAST>
__global__ __launch_bounds__(kBlock) void k_relbias_sums(const T* __restrict__ grad, const int64_t* __restrict__ q_at,
                                                          float* __restrict__ to, uint64_t by_head, uint64_t by_bucket,
                                                          unsigned buckets, unsigned tiles, Cut cut, Shape s, Buckets b) {
  __shared__ uint32_t border[kMostBuckets / 2 + 1];
  __shared__ float diagonal[kWaves][kMostRows + kCols];
  __shared__ float sums[kWaves][kMostBuckets];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint64_t head = blockIdx.y;
  fetch_borders(border, b);
  for (unsigned u = lane; u < buckets; u += 64) sums[wave][u] = 0.0f;
  __syncthreads();
  const unsigned tile = blockIdx.x * kWaves + wave;
  if (tile < tiles) {
    const Tile t(tile, cut, s);  // (of any head: cut.parts is 1)
    const Span<kWide> span(t.c0, lane, s.K);
    const T* from = grad + t.batch0 * s.in[0] + head * s.in[1] + t.r0 * s.in[2];
    const unsigned reach = (t.rows + kGroup - 1) / kGroup * kGroup;
    float high[kWide] = {};  // of the diagonals that begin the group's first row
    for (unsigned i = 0; i < t.rows; i += kGroup) {
      float sum[kGroup][kWide] = {};
      auto group = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        for (unsigned n = 0; n < t.batches; ++n) {
          Some<T, kWide> x[kGroup];
          span.template load<WHOLE, PAST>(x, from + n * s.in[0] + i * s.in[2], s.in[2], t.rows - i);
#pragma unroll
          for (unsigned r = 0; r < kGroup; ++r)
            if (WHOLE || i + r < t.rows)
#pragma unroll
              for (unsigned k = 0; k < kWide; ++k) sum[r][k] += x[r].at(k);
        }
      };
      if (i + kGroup <= t.rows)
        group(std::true_type());
      else
        group(std::false_type());
      float low[kWide] = {};
#pragma unroll
      for (unsigned r = 0; r < kGroup; ++r)
#pragma unroll
        for (unsigned k = 0; k < kWide; ++k) {
          if (k >= r)
            high[k - r] += sum[r][k];
          else
            low[kWide + k - r] += sum[r][k];
        }
#pragma unroll
      for (unsigned k = 0; k < kWide; ++k) {
        if (lane == 63) diagonal[wave][kCols - kWide + reach - i + k] = high[k];
        high[k] = low[k] + from_below(high[k], 0.0f);
      }
    }
#pragma unroll
    for (unsigned k = 0; k < kWide; ++k) diagonal[wave][lane * kWide + k] = high[k];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // diagonal[x] is the one that is x - reach columns to the right of the tile's corner
    const int32_t rel = nearer(s.rel0, q_at ? q_at[t.batch0] : 0, (int64_t)(t.c0 - t.r0 - reach));
    // (those that no element of the tile is on are left out)
    const unsigned reached = reach + (s.K - t.c0 < kCols ? (unsigned)(s.K - t.c0) : kCols);
    add_buckets(sums[wave], b, border, rel, 0, 64, reached, [&](unsigned x) { return diagonal[wave][x]; });
  }
  __syncthreads();
  put_sums(sums, to + head * by_head + blockIdx.x, by_bucket, buckets);
}

// Of narrow matrices: a workgroup sums a plane over its batches, and a lane each diagonal of the sums. An odd number of
// columns apart, the rows' elements that neighbouring diagonals begin with are in banks of their own.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_relbias_narrow_sums(const T* __restrict__ grad, const int64_t* __restrict__ q_at,
                                                                 float* __restrict__ to, uint64_t by_head, uint64_t by_bucket,
                                                                 unsigned buckets, Cut cut, Shape s, Buckets b) {
  constexpr unsigned kAhead = 4;  // batches asked for at a time
  __shared__ uint32_t border[kMostBuckets / 2 + 1];
  __shared__ float plane[kPlane];
  __shared__ float sums[kWaves][kMostBuckets];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint64_t head = blockIdx.y;
  fetch_borders(border, b);
  for (unsigned u = lane; u < buckets; u += 64) sums[wave][u] = 0.0f;
  const Tile t(blockIdx.x, cut, s);  // (of any head: cut.parts is 1)
  const Plane c(t.rows, (unsigned)s.K);
  const T* from = grad + t.batch0 * s.in[0] + head * s.in[1] + t.r0 * s.in[2];
  float sum[kEach] = {};
  auto some = [&](unsigned n0, auto count) {
    constexpr unsigned N = decltype(count)::value;
    T x[N][kEach];
#pragma unroll
    for (unsigned n = 0; n < N; ++n)
#pragma unroll
      for (unsigned i = 0; i < kEach; ++i)
        if (i < c.passes) x[n][i] = from[(n0 + n) * s.in[0] + c.row[i] * s.in[2] + c.col[i]];
#pragma unroll
    for (unsigned n = 0; n < N; ++n)
#pragma unroll
      for (unsigned i = 0; i < kEach; ++i)
        if (i < c.passes) sum[i] += (float)x[n][i];
  };
  unsigned n = 0;
  for (; n + kAhead <= t.batches; n += kAhead) some(n, std::integral_constant<unsigned, kAhead>());
  for (; n < t.batches; ++n) some(n, std::integral_constant<unsigned, 1>());
  const unsigned K = (unsigned)s.K, pitch = K | 1;
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (c.has(i)) plane[c.row[i] * pitch + c.col[i]] = sum[i];
  __syncthreads();
  // diagonal x begins at column x - (rows - 1) of row 0, or at column 0 of row rows - 1 - x
  const int32_t rel = nearer(s.rel0, q_at ? q_at[t.batch0] : 0, (int64_t)(0 - t.r0 - (t.rows - 1)));
  add_buckets(sums[wave], b, border, rel, wave * 64, kBlock, t.rows + K - 1, [&](unsigned x) {
    const unsigned r = x < t.rows ? t.rows - 1 - x : 0, k = x < t.rows ? 0 : x - (t.rows - 1);
    const unsigned cells = t.rows - r < K - k ? t.rows - r : K - k;
    const float* at = plane + r * pitch + k;
    float along = 0.0f;
#pragma unroll 8
    for (unsigned i = 0; i < cells; ++i) along += at[i * (pitch + 1)];
    return along;
  });
  __syncthreads();
  put_sums(sums, to + head * by_head + blockIdx.x, by_bucket, buckets);
}

// The workgroups' sums of a bucket and head: a wavefront to each.
__global__ __launch_bounds__(64) void k_relbias_join(const float* __restrict__ partial, unsigned buckets, unsigned slots, uint64_t H,
                                                      float* __restrict__ grad_table) {
  const uint64_t head = blockIdx.y;
  const unsigned u = blockIdx.x;
  const float* from = partial + (head * buckets + u) * slots;
  float sum = 0.0f;
  for (unsigned i = threadIdx.x; i < slots; i += 64) sum += from[i];
  sum = sum_along(sum, 0);
  if (threadIdx.x == 63) grad_table[(uint64_t)u * H + head] = sum;
}

// --- the host's checks -------------------------------------------------------------------------------------------

int check(int type, size_t H, size_t B, size_t Q, size_t K, int64_t q_first, int64_t k_first) {
  if (!type_bytes(type)) return set_error(PSKV_EINVAL, "type %d: PSKV_F32, PSKV_F16 or PSKV_BF16", type);
  if (H == 0 || H > 65535) return set_error(PSKV_EINVAL, "1 to 65535 heads");
  if (B > (1u << 20) || Q > (1u << 20) || K > (1u << 30)) return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
  const int64_t most = 1ll << 60;
  if (q_first > most || q_first < -most || k_first > most || k_first < -most)
    return set_error(PSKV_EINVAL, "positions beyond 2^60");
  return PSKV_OK;
}

int buckets_or_error(Buckets* b, size_t buckets, uint64_t max_distance, int two_sided) {
  bool ok = false;
  try {
    ok = make_buckets(b, buckets, max_distance, two_sided != 0);
  } catch (const std::bad_alloc&) {
    return set_error(PSKV_ENOMEM, "no memory for the borders of the buckets");
  }
  if (!ok)
    return set_error(PSKV_EINVAL, "%zu buckets up to distance %llu: 2 (two-sided 4) to %u buckets, and a distance beyond those with "
                     "a bucket of their own, up to 2^30", buckets, (unsigned long long)max_distance, kMostBuckets);
  return PSKV_OK;
}

// The bytes from the first element of a [B, H, Q, K] tensor to behind its last.
uint64_t extent(const int64_t* stride, const Shape& s, size_t size) {
  return ((s.B - 1) * (uint64_t)stride[0] + (s.H - 1) * (uint64_t)stride[1] + (s.Q - 1) * (uint64_t)stride[2] + s.K) * size;
}

// Whether a stretch of memory shares a byte with a [B, H, Q, K] tensor.
bool lies_in(const void* at, uint64_t bytes, const void* tensor, const int64_t* stride, const Shape& s, size_t size) {
  Nest dim[3] = {{s.B, (uint64_t)stride[0] * size}, {s.H, (uint64_t)stride[1] * size}, {s.Q, (uint64_t)stride[2] * size}};
  std::sort(dim, dim + 3, [](const Nest& a, const Nest& b) { return a.stride > b.stride; });
  const uint64_t first = reinterpret_cast<uintptr_t>(at);
  return touches(first, first + bytes, reinterpret_cast<uintptr_t>(tensor), dim, 3, s.K * size);
}

int check_strides(const char* what, const int64_t* stride, const Shape& s, bool written) {
  if (!stride) return set_error(PSKV_EINVAL, "%s: no strides", what);
  uint64_t n[4] = {s.B, s.H, s.Q, s.K}, by[4] = {(uint64_t)stride[0], (uint64_t)stride[1], (uint64_t)stride[2], 1};
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] > (1ll << 40)) return set_error(PSKV_EINVAL, "%s: strides of 0 to 2^40", what);
  if (!written) return PSKV_OK;
  // every element has a place of its own: the next wider stride begins behind what the narrower ones reach
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (by[j] < by[i] || (by[j] == by[i] && n[j] < n[i])) {
        const uint64_t x = by[i], y = n[i];
        by[i] = by[j], n[i] = n[j];
        by[j] = x, n[j] = y;
      }
  uint64_t reach = 0;
  for (int i = 0; i < 4; ++i) {
    if (n[i] < 2) continue;
    if (by[i] <= reach) return set_error(PSKV_EINVAL, "%s: elements that are written lie upon each other", what);
    reach += (n[i] - 1) * by[i];
  }
  return PSKV_OK;
}

constexpr uint64_t kFilled = 2048;  // wavefronts that fill the GPU

// Of the bias: a wavefront takes eight rows, so that those at work stay close together in memory. Where there is one query only, heads are put
// together by two, up to eight, as long as there are wavefronts enough to fill the GPU before: half as many may be left (64 x 16 x 4,096 bf16:
// 1,024, of eight heads).
Cut cut_for_bias(size_t B, size_t H, size_t Q, size_t K, size_t size) {
  Cut c{};
  c.cols = 64 * 16 / (unsigned)size;
  c.rows = kGroup;
  c.across = (unsigned)((K + c.cols - 1) / c.cols);
  c.strips = (unsigned)((Q + c.rows - 1) / c.rows);
  c.batches = c.heads = 1;
  c.chunks = (unsigned)B;
  c.parts = (unsigned)H;
  while (Q == 1 && c.heads < kGroup && c.heads < H && c.tiles() >= kFilled) {
    c.heads *= 2;
    c.parts = (unsigned)((H + c.heads - 1) / c.heads);
  }
  return c;
}

// Of either: the planes of narrow matrices, for as many batches as there are workgroups without to fill the GPU.
Cut cut_for_planes(size_t B, size_t heads, size_t Q, size_t K, bool own_positions) {
  Cut c{};
  c.cols = (unsigned)K;
  c.rows = (unsigned)plane_rows(Q, K);
  c.across = c.heads = c.parts = 1;
  c.strips = (unsigned)((Q + c.rows - 1) / c.rows);
  c.batches = own_positions ? 1 : (unsigned)B;
  for (;;) {
    c.chunks = (unsigned)((B + c.batches - 1) / c.batches);
    if (c.batches == 1 || c.tiles() * heads >= kFilled) return c;
    c.batches = (c.batches + 1) / 2;
  }
}

// Of the gradient: the tiles of a head. Enough wavefronts to fill the GPU, if that can be had: fewer rows for each first, then fewer
// batches, then fewer rows again (64 rows as long as there are batches to share out: 16 x 2048 x 2048 bf16 28 us, from 32 rows on 32).
Cut cut_for_sums(size_t B, size_t H, size_t Q, size_t K, bool own_positions) {
  Cut c{};
  c.cols = kCols;
  c.rows = kMostRows;
  while (c.rows / 2 >= Q && c.rows > kGroup) c.rows /= 2;
  c.batches = own_positions ? 1 : (unsigned)B;
  c.across = (unsigned)((K + kCols - 1) / kCols);
  c.heads = c.parts = 1;
  for (;;) {
    c.strips = (unsigned)((Q + c.rows - 1) / c.rows);
    c.chunks = (unsigned)((B + c.batches - 1) / c.batches);
    if (c.tiles() * H >= kFilled) break;
    if (c.rows > 64)
      c.rows /= 2;
    else if (c.batches > 1)
      c.batches = (c.batches + 1) / 2;
    else if (c.rows > kGroup)
      c.rows /= 2;
    else
      break;
  }
  return c;
}

// How the gradient is cut up, and the workgroups of a head.
struct SumsCut {
  bool narrow;
  Cut cut;
  uint64_t groups;
  SumsCut(size_t B, size_t H, size_t Q, size_t K, bool own_positions) : narrow(sums_by_planes(Q, K, own_positions)) {
    if (narrow) {
      cut = cut_for_planes(B, H, Q, K, own_positions);
      groups = cut.tiles();
      narrow = groups <= 1u << 20;  // (beyond, smaller working memory counts)
    }
    if (!narrow) {
      cut = cut_for_sums(B, H, Q, K, own_positions);
      groups = (cut.tiles() + kWaves - 1) / kWaves;
    }
  }
};

}  // namespace
}  // namespace pskv

using namespace pskv;

static_assert(kMostBuckets == PSKV_RELBIAS_MAX_BUCKETS, "the header says so");

extern "C" int pskv_relbias_bucket(int64_t rel, size_t buckets, uint64_t max_distance, int two_sided) {
  clear_error();
  Buckets b;
  const int rc = buckets_or_error(&b, buckets, max_distance, two_sided);
  return rc ? rc : (int)bucket_of(b, b.border, nearer(rel));
}

extern "C" int pskv_relbias(int device, void* stream, int type, const float* table, size_t buckets, size_t H,
                            uint64_t max_distance, int two_sided, int64_t q_first, int64_t k_first, const int64_t* q_at,
                            const void* scores, const int64_t* scores_stride, void* out, const int64_t* out_stride, size_t B,
                            size_t Q, size_t K) {
  clear_error();
  int rc = check(type, H, B, Q, K, q_first, k_first);
  if (rc) return rc;
  Buckets b;
  if ((rc = buckets_or_error(&b, buckets, max_distance, two_sided))) return rc;
  if (B == 0 || Q == 0 || K == 0) return PSKV_OK;
  if (!table || !out) return set_error(PSKV_EINVAL, "null buffer");
  Shape s{B, H, Q, K, k_first - q_first, {0, 0, 0}, {0, 0, 0}};
  if ((rc = check_strides("out", out_stride, s, true))) return rc;
  if (scores && (rc = check_strides("scores", scores_stride, s, false))) return rc;
  for (int i = 0; i < 3; ++i) {
    s.out[i] = (uint64_t)out_stride[i];
    s.in[i] = scores ? (uint64_t)scores_stride[i] : 0;
  }
  const uint64_t out_bytes = extent(out_stride, s, type_bytes(type));
  if (overlap(table, buckets * H * sizeof(float), out, out_bytes) || (q_at && overlap(q_at, B * sizeof(int64_t), out, out_bytes)))
    return set_error(PSKV_EINVAL, "out overlaps the table or the positions");
  if (scores) {
    const uint64_t a = reinterpret_cast<uintptr_t>(scores), o = reinterpret_cast<uintptr_t>(out), size = type_bytes(type);
    bool same = a == o;
    const size_t n[3] = {B, H, Q};
    for (int i = 0; i < 3; ++i) same = same && (n[i] < 2 || s.in[i] == s.out[i]);
    if (!same && a < o + out_bytes && o < a + extent(scores_stride, s, size))
      return set_error(PSKV_EINVAL, "out lies in the scores and is not the same tensor");
  }
  const bool narrow = by_planes(Q, K, type_bytes(type), scores != nullptr, q_at != nullptr);
  Cut cut = narrow ? cut_for_planes(B, H, Q, K, q_at != nullptr) : cut_for_bias(B, H, Q, K, type_bytes(type));
  if (narrow) cut.heads = 1, cut.parts = (unsigned)H;
  if (cut.tiles() > kMostTiles) return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(grid_for(cut.tiles(), narrow ? 1 : kWaves, 1u << 22)), dim3(kBlock), 0, static_cast<hipStream_t>(stream),
                         table, q_at, static_cast<const T*>(scores), static_cast<T*>(out), (unsigned)cut.tiles(), cut, s, b);
    };
    if (narrow)
      launch(scores ? k_relbias_narrow<T, true> : k_relbias_narrow<T, false>);
    else if (Q == 1)
      launch(scores ? k_relbias_step<T, true> : k_relbias_step<T, false>);
    else if (B * H * Q * K * sizeof(T) * (scores ? 2 : 1) > kPastBytes)
      launch(scores ? k_relbias<T, true, true> : k_relbias<T, false, true>);
    else
      launch(scores ? k_relbias<T, true, false> : k_relbias<T, false, false>);
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}

extern "C" size_t pskv_relbias_grad_room(size_t buckets, size_t H, size_t B, size_t Q, size_t K, int own_positions) {
  if (B == 0 || Q == 0 || K == 0 || B > (1u << 20) || Q > (1u << 20) || K > (1u << 30)) return 0;
  const uint64_t groups = SumsCut(B, H, Q, K, own_positions != 0).groups;
  return groups == 1 ? 0 : groups * buckets * H * sizeof(float);
}

extern "C" int pskv_relbias_grad(int device, void* stream, int type, const void* grad, const int64_t* grad_stride,
                                 size_t buckets, size_t H, uint64_t max_distance, int two_sided, int64_t q_first,
                                 int64_t k_first, const int64_t* q_at, size_t B, size_t Q, size_t K, float* grad_table,
                                 void* work, size_t work_bytes) {
  clear_error();
  int rc = check(type, H, B, Q, K, q_first, k_first);
  if (rc) return rc;
  Buckets b;
  if ((rc = buckets_or_error(&b, buckets, max_distance, two_sided))) return rc;
  if (!grad_table) return set_error(PSKV_EINVAL, "null buffer");
  Shape s{B, H, Q, K, k_first - q_first, {0, 0, 0}, {0, 0, 0}};
  const bool any = B && Q && K;
  bool narrow = false;
  Cut cut{};
  uint64_t groups = 0;
  if (!any) work = nullptr;  // (nothing is summed up, and there are no strides)
  if (any) {
    if (!grad) return set_error(PSKV_EINVAL, "null buffer");
    if ((rc = check_strides("grad", grad_stride, s, false))) return rc;
    for (int i = 0; i < 3; ++i) s.in[i] = (uint64_t)grad_stride[i];
    const SumsCut sums(B, H, Q, K, q_at != nullptr);
    narrow = sums.narrow;
    cut = sums.cut;
    groups = sums.groups;
    if (groups > kMostTiles / kBlock) return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
    const size_t room = groups == 1 ? 0 : groups * buckets * H * sizeof(float);
    if (room == 0)
      work = nullptr;
    else if (!work || work_bytes < room || (reinterpret_cast<uintptr_t>(work) & 3))
      return set_error(PSKV_EINVAL, "this gradient takes %zu bytes of working memory, %zu given", room, work ? work_bytes : (size_t)0);
  }
  const uint64_t table_bytes = buckets * H * sizeof(float), used = work ? groups * table_bytes : 0;
  if (any && lies_in(grad_table, table_bytes, grad, grad_stride, s, type_bytes(type)))
    return set_error(PSKV_EINVAL, "the gradient of the table lies in the gradient that is read");
  if (any && q_at && (overlap(q_at, B * sizeof(int64_t), grad_table, table_bytes) || overlap(q_at, B * sizeof(int64_t), work, used)))
    return set_error(PSKV_EINVAL, "the gradient of the table or the working memory overlaps the positions");
  if (work && (overlap(work, used, grad_table, table_bytes) ||
              overlap(work, used, grad, extent(grad_stride, s, type_bytes(type)))))
    return set_error(PSKV_EINVAL, "the working memory overlaps the gradients");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* partial = static_cast<float*>(work);
  if (any)
    with_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      auto launch = [&](auto kernel, auto... tiles) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups, (unsigned)H), dim3(kBlock), 0, st, static_cast<const T*>(grad), q_at,
                           groups == 1 ? grad_table : partial, groups == 1 ? (uint64_t)1 : buckets * groups,
                           groups == 1 ? (uint64_t)H : groups, (unsigned)buckets, tiles..., cut, s, b);
      };
      // (of several gradients of 83 MB in turn, 31 us each, some is still in the memory-side cache, 34 past it; of 134 MB 32 and 29)
      if (narrow)
        launch(k_relbias_narrow_sums<T>);
      else if (B * H * Q * K * sizeof(T) > kPastBytes / 2)
        launch(k_relbias_sums<T, true>, (unsigned)cut.tiles());
      else
        launch(k_relbias_sums<T, false>, (unsigned)cut.tiles());
    });
  if (groups != 1)
    hipLaunchKernelGGL(k_relbias_join, dim3((unsigned)buckets, (unsigned)H), dim3(64), 0, st, partial, (unsigned)buckets,
                       (unsigned)groups, (uint64_t)H, grad_table);
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}
