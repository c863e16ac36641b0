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

}  // namespace pskv
#endif  // PSKV_ROW_TYPES_H_
