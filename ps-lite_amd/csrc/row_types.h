// What the operators on rows share: the types an element may have and vectors of them at any address.
#ifndef PSKV_ROW_TYPES_H_
#define PSKV_ROW_TYPES_H_
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pskv/capi.h"
#include "row_span.h"

namespace pskv {

// 16 bytes of a row. Rows may begin at any element (odd lengths, slices of columns), so a vector is aligned to its elements
// only: the GPU takes such accesses as they are, in one instruction.
template <typename T>
struct Row {
  static constexpr int kWide = 16 / (int)sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A vector at p, by an access that stays in the caches or by one that goes past them (what nobody reads again soon).
template <bool PAST, typename T>
__device__ __forceinline__ typename Row<T>::Vec get(const T* p) {
  const typename Row<T>::Vec* at = reinterpret_cast<const typename Row<T>::Vec*>(p);
  return PAST ? __builtin_nontemporal_load(at) : *at;
}
template <bool PAST, typename T>
__device__ __forceinline__ void put(T* p, typename Row<T>::Vec v) {
  typename Row<T>::Vec* at = reinterpret_cast<typename Row<T>::Vec*>(p);
  if (PAST)
    __builtin_nontemporal_store(v, at);
  else
    *at = v;
}

inline size_t type_bytes(int type) { return type == PSKV_F32 ? 4 : type == PSKV_F16 || type == PSKV_BF16 ? 2 : 0; }

// Calls f with a null pointer of the element type that `type` (one that type_bytes knows) names.
template <typename F>
inline void with_type(int type, F f) {
  if (type == PSKV_F32)
    f(static_cast<float*>(nullptr));
  else if (type == PSKV_F16)
    f(static_cast<_Float16*>(nullptr));
  else
    f(static_cast<__bf16*>(nullptr));
}

// Calls f with std::true_type or std::false_type.
template <typename F>
inline void with_flag(bool flag, F f) {
  if (flag)
    f(std::true_type());
  else
    f(std::false_type());
}

// What moves more than so many bytes, the size of the memory-side cache, does not stay there anyway.
constexpr uint64_t kPastBytes = 256u << 20;

}  // namespace pskv
#endif  // PSKV_ROW_TYPES_H_
