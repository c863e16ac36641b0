// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3"
// (2011): four words from a counter of four and a key of two, by ten rounds of two products each.
#ifndef PSKV_PHILOX_H_
#define PSKV_PHILOX_H_
#include <stdint.h>

#ifdef __HIP__
#define PSKV_PHILOX_FN __host__ __device__ __forceinline__
#else
#define PSKV_PHILOX_FN inline
#endif

namespace pskv {

// (one instruction on the GPU, which the compiler does not choose by itself)
PSKV_PHILOX_FN uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
#else
  return a ^ b ^ c;
#endif
}

struct Drawn {
  uint32_t word[4];
};

PSKV_PHILOX_FN Drawn philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Drawn{{c0, c1, c2, c3}};
}

}  // namespace pskv
#endif  // PSKV_PHILOX_H_
