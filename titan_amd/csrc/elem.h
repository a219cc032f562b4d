// Element types of the kernels that take more than one, and vectors of them.
#pragma once

#include "common.h"

template <int DT>
struct Elem;
template <>
struct Elem<QMOE_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float load(T v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ T store(float f) { return (T)f32_to_bf16(f); }
};
template <>
struct Elem<QMOE_FP16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float load(T v) { return (float)v; }
  static __device__ __forceinline__ T store(float f) { return (_Float16)f; }
};
template <>
struct Elem<QMOE_FP32> {
  typedef float T;
  static __device__ __forceinline__ float load(T v) { return v; }
  static __device__ __forceinline__ T store(float f) { return f; }
};

// N consecutive elements, moved as one access of N * sizeof(T) bytes.
template <typename T, int N>
struct Vec {
  typedef T V __attribute__((ext_vector_type(N)));
};
template <typename T>
struct Vec<T, 1> {
  typedef T V;
};
template <typename T, int N>
__device__ __forceinline__ T at(const typename Vec<T, N>::V& v, int i) {
  if constexpr (N == 1) return v;
  else return v[i];
}
template <typename T, int N>
__device__ __forceinline__ void set(typename Vec<T, N>::V& v, int i, T x) {
  if constexpr (N == 1) v = x;
  else v[i] = x;
}

namespace qmoe {
// Bytes of an element, 0 for a type that there is none of.
inline int size_of(int dtype) { return dtype == QMOE_FP32 ? 4 : dtype == QMOE_BF16 || dtype == QMOE_FP16 ? 2 : 0; }
}  // namespace qmoe
