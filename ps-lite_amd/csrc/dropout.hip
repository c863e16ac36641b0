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

template <typename T, bool FEW>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* x, T* out, const uint64_t* __restrict__ keys, uint64_t first,
                                                     const uint64_t* __restrict__ step, uint64_t seed, uint64_t n, uint64_t k,
                                                     uint64_t x_stride, uint64_t out_stride, unsigned least, float scale, Divisor per_row) {
  using Vec = typename Row<T>::Vec;
  constexpr unsigned W = Row<T>::kWide;
  if (step) seed += *step;
  const uint64_t blocks = (k + kDrawn - 1) / kDrawn;
  for (uint64_t at = (uint64_t)blockIdx.x * kBlock + threadIdx.x; at < n * blocks; at += (uint64_t)gridDim.x * kBlock) {
    const uint64_t r = FEW ? per_row.of((uint32_t)at) : at / blocks, q = at - r * blocks;
    const uint64_t key = keys ? keys[r] : first + r;
    const Drawn d = philox((uint32_t)key, (uint32_t)(key >> 32), (uint32_t)q, 0, (uint32_t)seed, (uint32_t)(seed >> 32));
    const T* from = x + r * x_stride + q * kDrawn;
    T* to = out + r * out_stride + q * kDrawn;
    const unsigned wide = k - q * kDrawn < kDrawn ? (unsigned)(k - q * kDrawn) : kDrawn;
    auto kept = [&](unsigned i, T v) {
      const unsigned bits = i & 1 ? d.word[i / 2] >> 16 : d.word[i / 2] & 0xffffu;
      return bits >= least ? (T)((float)v * scale) : (T)0.0f;
    };
    if (wide == kDrawn) {
#pragma unroll
      for (unsigned i = 0; i < kDrawn; i += W) {
        const Vec v = *reinterpret_cast<const Vec*>(from + i);
        Vec o;
#pragma unroll
        for (unsigned e = 0; e < W; ++e) o[e] = kept(i + e, v[e]);
        *reinterpret_cast<Vec*>(to + i) = o;
      }
    } else {
#pragma unroll
      for (unsigned i = 0; i < kDrawn; ++i)
        if (i < wide) to[i] = kept(i, from[i]);
    }
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
  if (!in_place && rows_overlap({x, n, k, x_stride, size}, {out, n, k, out_stride, size}))
    return set_error(PSKV_EINVAL, "out overlaps x and is not the same rows");
  const unsigned least = (unsigned)floor(p * 65536.0 + 0.5);
  const float scale = least < 65536 ? (float)(65536.0 / (65536 - least)) : 0.0f;
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto kernel = n * blocks < (1ull << 32) ? k_dropout<T, true> : k_dropout<T, false>;
    hipLaunchKernelGGL(kernel, dim3(grid_for(n * blocks, kBlock, 1u << 22)), dim3(kBlock), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T*>(x), static_cast<T*>(out), keys, first, step, seed, (uint64_t)n, (uint64_t)k,
                       (uint64_t)x_stride, (uint64_t)out_stride, least, scale, Divisor((uint32_t)blocks));
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}
