// Dropout of rows without a stored mask (gfx950): whether an element stays is drawn from its row's key and its column, so the
// gradient's call draws the same again, in whatever order its rows come.
//     words = Philox4x32-10(key: seed, counter: row key low, high, column / 8, 0), 16 bits of them for each of 8 columns
//     y = bits >= least ? x * 65536 / (65536 - least) : 0,   least = round(65536 p)
// Sixteen bits an element: one draw of ten rounds serves 8 elements; with 32 bits the rounds, not the memory, would be what
// bounds rows of 16-bit elements. The share that is dropped is least / 65536, at most 2^-17 from p, and the scale goes by it.
#include <hip/hip_runtime.h>
#include <math.h>

#include "host_common.h"
#include "philox.h"
#include "row_types.h"

namespace pskv {
namespace {

constexpr unsigned kBlock = 256;
constexpr unsigned kDrawn = 8;  // columns that one draw serves
constexpr uint64_t kMostDraws = (1ull << 31) - 2 * kBlock;  // of a launch

template <typename T>
__device__ __forceinline__ T keep(uint32_t word, bool high, unsigned least, T v, float scale) {
  return (high ? word >> 16 : word & 0xffffu) >= least ? (T)((float)v * scale) : (T)0.0f;
}

// n / d for n below 2^32 by a product (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divisor {
  uint32_t d, magic, shift;
  explicit Divisor(uint32_t by) : d(by), magic(0), shift(0) {
    unsigned l = 0;
    while (l < 32 && (1ull << l) < by) ++l;
    magic = (uint32_t)(((((1ull << l) - by) << 32) / by) + 1);
    shift = l;
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const {
    const uint32_t t = __umulhi(magic, n);
    return shift == 0 ? n : (t + ((n - t) >> 1)) >> (shift - 1);
  }
};

// 16-bit types: a lane takes the 8 columns of a draw, 16 bytes. Indexes are those of draws. The ten rounds' products (16 cycles each)
// and the memory take about the same time: 65,536 rows of 2,048 bf16 in 90 us, 6.0 TB/s; 4,099 of 1,001 in 5.9 to 6.4 us.
template <typename T, bool PAST>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* x, T* out, const uint64_t* __restrict__ keys, uint64_t first,
                                                     const uint64_t* __restrict__ step, uint64_t seed, uint32_t draws, uint32_t k,
                                                     uint64_t x_stride, uint64_t out_stride, unsigned least, float scale,
                                                     Divisor per_row) {
  constexpr unsigned W = Row<T>::kWide;
  static_assert(W == kDrawn, "a vector is what a draw serves");
  if (step) seed += *step;
  const uint32_t at = blockIdx.x * kBlock + threadIdx.x;
  if (at >= draws) return;
  const uint32_t r = per_row.of(at), q = at - r * per_row.d;
  const uint64_t key = keys ? keys[r] : first + r;
  const uint32_t c = q * kDrawn;
  const Drawn d = philox((uint32_t)key, (uint32_t)(key >> 32), q, 0, (uint32_t)seed, (uint32_t)(seed >> 32));
  const T* from = x + r * x_stride + c;
  T* to = out + r * out_stride + c;
  auto kept = [&](unsigned i, T v) { return keep(d.word[i / 2], i & 1, least, v, scale); };
  if (k - c >= kDrawn) {
    const typename Row<T>::Vec v = get<PAST>(from);
    typename Row<T>::Vec o;
#pragma unroll
    for (unsigned i = 0; i < kDrawn; ++i) o[i] = kept(i, v[i]);
    put<PAST>(to, o);
  } else {
#pragma unroll
    for (unsigned i = 0; i < kDrawn; ++i)
      if (i < k - c) to[i] = kept(i, from[i]);
  }
}

__device__ __forceinline__ uint32_t of_neighbour(uint32_t v) {  // lanes 2i and 2i + 1 exchange
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1 /* quad_perm:[1,0,3,2] */, 0xf, 0xf, false);
}

// float32: a draw's 8 columns are 32 bytes, and lanes that each take 32 bytes leave every access half of its lines. So a lane
// takes four columns here and four 64 lanes further on; of two neighbours the even one draws for both here, the odd one there,
// and they exchange halves. Indexes are those of quads of columns, two to a draw. 1M rows of 64: 80 us, 6.5 TB/s, past the caches
// (32 bytes to a lane: 100, and 237 past the caches; every lane drawing for its four columns: 109).
template <bool PAST>
__global__ __launch_bounds__(kBlock) void k_dropout_pairs(const float* x, float* out, const uint64_t* __restrict__ keys, uint64_t first,
                                                           const uint64_t* __restrict__ step, uint64_t seed, uint32_t quads, uint32_t k,
                                                           uint64_t x_stride, uint64_t out_stride, unsigned least, float scale,
                                                           Divisor per_row) {
  using Vec = Row<float>::Vec;
  if (step) seed += *step;
  const unsigned lane = threadIdx.x & 63;
  const bool odd = lane & 1;
  const uint32_t here = (blockIdx.x * kBlock + threadIdx.x - lane) * 2 + lane;
  const uint32_t mine = odd ? here + 64 : here;
  const uint32_t r = per_row.of(mine), q = mine - r * per_row.d;
  uint64_t key = first + r;
  if (keys && mine < quads) key = keys[r];
  const Drawn d = philox((uint32_t)key, (uint32_t)(key >> 32), q >> 1, 0, (uint32_t)seed, (uint32_t)(seed >> 32));
  const uint32_t other0 = of_neighbour(odd ? d.word[0] : d.word[2]), other1 = of_neighbour(odd ? d.word[1] : d.word[3]);
  const uint32_t other_r = of_neighbour(r), other_q = of_neighbour(q);
  // (the lower half of the draw is the even lane's)
  const uint32_t rows[2] = {odd ? other_r : r, odd ? r : other_r};
  const uint32_t cols[2] = {(((odd ? other_q : q) & ~1u) + (odd ? 1 : 0)) * 4, (((odd ? q : other_q) & ~1u) + (odd ? 1 : 0)) * 4};
  const uint32_t words[2][2] = {{odd ? other0 : d.word[0], odd ? other1 : d.word[1]}, {odd ? d.word[2] : other0, odd ? d.word[3] : other1}};
  Vec v[2];
  bool whole[2];
#pragma unroll
  for (unsigned h = 0; h < 2; ++h) {
    const bool is = here + h * 64 < quads && cols[h] < k;
    whole[h] = is && k - cols[h] >= 4;
    const float* from = x + rows[h] * x_stride + cols[h];
    if (whole[h]) v[h] = get<PAST>(from);
    if (is && !whole[h]) {
      float* to = out + rows[h] * out_stride + cols[h];
#pragma unroll
      for (unsigned i = 0; i < 3; ++i)
        if (i < k - cols[h]) to[i] = keep(words[h][i / 2], i & 1, least, from[i], scale);
    }
  }
#pragma unroll
  for (unsigned h = 0; h < 2; ++h) {
    Vec o;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) o[i] = keep(words[h][i / 2], i & 1, least, v[h][i], scale);
    if (whole[h]) put<PAST>(out + rows[h] * out_stride + cols[h], o);
  }
}

}  // namespace
}  // namespace pskv

using namespace pskv;

extern "C" int pskv_dropout(int device, void* stream, int type, const void* x, size_t x_stride, void* out, size_t out_stride,
                            size_t n, size_t k, double p, uint64_t seed, const uint64_t* step, const uint64_t* keys,
                            uint64_t first) {
  clear_error();
  const size_t size = type_bytes(type);
  if (!size) return set_error(PSKV_EINVAL, "type %d: PSKV_F32, PSKV_F16 or PSKV_BF16", type);
  if (!(p >= 0.0 && p <= 1.0)) return set_error(PSKV_EINVAL, "p = %g is no probability", p);
  if (keys && first) return set_error(PSKV_EINVAL, "rows are counted by their keys or from a first number, not both");
  if (k > (1ull << 30) || n > (1ull << 40) || (n && k > (1ull << 42) / n))
    return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
  if (n == 0 || k == 0) return PSKV_OK;
  if (x_stride > (1ull << 40) || out_stride > (1ull << 40)) return set_error(PSKV_EINVAL, "rows 2^40 elements apart at most");
  if (n > 1 && out_stride < k) return set_error(PSKV_EINVAL, "out: rows that are written lie upon each other");
  if (!x || !out) return set_error(PSKV_EINVAL, "null buffer");
  const uint64_t blocks = (k + kDrawn - 1) / kDrawn;
  const bool in_place = x == out && (n == 1 || x_stride == out_stride);
  const RowSpan to{out, n, k, out_stride, size};
  if (!in_place && rows_overlap({x, n, k, x_stride, size}, to))
    return set_error(PSKV_EINVAL, "out overlaps x and is not the same rows");
  if (rows_overlap(stretch(keys, n * sizeof(uint64_t)), to) || rows_overlap(stretch(step, sizeof(uint64_t)), to))
    return set_error(PSKV_EINVAL, "out overlaps the keys or the step");
  const unsigned least = (unsigned)floor(p * 65536.0 + 0.5);
  const float scale = least < 65536 ? (float)(65536.0 / (65536 - least)) : 0.0f;
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // (a launch counts its draws in 31 bits)
  const uint64_t most = kMostDraws / blocks;
  for (uint64_t r0 = 0; r0 < n; r0 += most) {
    const uint64_t rows = n - r0 < most ? n - r0 : most;
    const uint32_t draws = (uint32_t)(rows * blocks);
    const dim3 grid((draws + kBlock - 1) / kBlock);
    const uint64_t* some = keys ? keys + r0 : nullptr;
    with_flag(2 * n * k * size > kPastBytes, [&](auto far) {
      constexpr bool PAST = decltype(far)::value;
      with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const T* from = static_cast<const T*>(x) + r0 * x_stride;
        T* to = static_cast<T*>(out) + r0 * out_stride;
        if constexpr (sizeof(T) == 4)
          hipLaunchKernelGGL(k_dropout_pairs<PAST>, grid, dim3(kBlock), 0, st, from, to, some, first + r0, step, seed, 2 * draws,
                             (uint32_t)k, (uint64_t)x_stride, (uint64_t)out_stride, least, scale, Divisor((uint32_t)(2 * blocks)));
        else
          hipLaunchKernelGGL((k_dropout<T, PAST>), grid, dim3(kBlock), 0, st, from, to, some, first + r0, step, seed, draws, (uint32_t)k,
                             (uint64_t)x_stride, (uint64_t)out_stride, least, scale, Divisor((uint32_t)blocks));
      });
    });
    PSKV_HIP(hipGetLastError());
  }
  return PSKV_OK;
}
