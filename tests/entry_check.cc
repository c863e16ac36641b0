// Entry points of the position bias as plain host code, unoptimized, with a runtime that has no device: what they look at before they
// select one. Prints what a gradient of [B, Q, K] returns that is given working memory and no strides.
#include "../ps-lite_amd/csrc/relbias.hip"

#include <stdio.h>
#include <stdlib.h>

namespace pskv {
int set_error(int code, const char*, ...) { return code; }
void clear_error() {}
}  // namespace pskv

extern "C" {
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipErrorInvalidDevice; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return ""; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { abort(); }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { abort(); }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { abort(); }
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipUnregisterFatBinary(void**) {}
}

int main(int, char** at) {
  float table[32 * 4], work[64];
  const size_t B = atoi(at[1]), Q = atoi(at[2]), K = atoi(at[3]);
  printf("%d\n", pskv_relbias_grad(1, nullptr, PSKV_F32, nullptr, nullptr, 32, 4, 128, 1, 0, 0, nullptr, B, Q, K, table, work, sizeof work));
  return 0;
}
