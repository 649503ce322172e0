// Helpers shared by the sequence encoder's kernels (attention.hip, norm.hip,
// dropout.hip): element types, vectors of them and alignment.
#pragma once

#include "common.h"

// short vectors of an element type (float, _Float16, __bf16)
template <typename T>
struct chain_vec {
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef T v8 __attribute__((ext_vector_type(8)));
};
template <typename T>
using v4 = typename chain_vec<T>::v4;
template <typename T>
using v8 = typename chain_vec<T>::v8;
typedef float f32x16 __attribute__((ext_vector_type(16)));

// true for NULL, too: an absent operand does not restrict the vector path
static inline bool chain_aligned16(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
