// Helpers shared by the sequence encoders' kernels (attention.hip, norm.hip,
// dropout.hip, delta.h, rmsnorm.hip, embedding.hip): element types, vectors of
// them and alignment.
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

// 8 elements that are aligned as one, and 8 channels of a row from el on, in fp32
template <typename T>
struct loose8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x8 load_row8(const T* row, int el, int width) {
  f32x8 x{};
  if (el + 8 <= width) {
    x = __builtin_convertvector(*reinterpret_cast<const typename loose8<T>::type*>(row + el),
                                f32x8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (el + j < width) x[j] = (float)row[el + j];
  }
  return x;
}
template <typename T>
__device__ __forceinline__ void store_row8(T* row, int el, int width, f32x8 x) {
  if (el + 8 <= width) {
    *reinterpret_cast<typename loose8<T>::type*>(row + el) =
        __builtin_convertvector(x, typename loose8<T>::type);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (el + j < width) row[el + j] = (T)x[j];
  }
}

// A grid of `groups` x `parts` workgroups of 256 threads.  An axis holds fewer than
// 2^32 threads and drops those above without an error: what is over goes on along z,
// where workgroups past the last one do nothing.
static inline dim3 chain_grid(int64_t groups, unsigned parts = 1) {
  constexpr int64_t most = int64_t(1) << 23;
  if (groups <= most) return dim3((unsigned)groups, parts);
  return dim3((unsigned)most, parts, mlcg_div_up(groups, most));
}
__device__ __forceinline__ int64_t chain_group() {
  return blockIdx.x + (int64_t)blockIdx.z * gridDim.x;
}

// true for NULL, too: an absent operand does not restrict the vector path
static inline bool chain_aligned16(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
