// Values to 8-bit codes and their row's scale, and accesses of rows that begin
// at any element's address (format in int8_rows.hip).
#pragma once

#include "elem.h"

namespace qmoe_i8 {

// Larger |v| have larger bits, infinities and NaN the largest.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kInfinite = 0x7F800000u;

__device__ __forceinline__ int code_of(float v, float s) {
  if (!(s > 0.f)) return 0;
  return (int)fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.f), 127.f);
}
__device__ __forceinline__ float scale_of(uint32_t top) {
  return top >= kInfinite ? __uint_as_float(0x7FC00000u) : __fdiv_rn(__uint_as_float(top), 127.f);
}

// N elements at any element's address.
template <class T, int N>
struct __attribute__((packed)) Loose {
  typename Vec<T, N>::V v __attribute__((aligned(1)));
};
template <class T, int N>
__device__ __forceinline__ typename Vec<T, N>::V get(const T* p) {
  return reinterpret_cast<const Loose<T, N>*>(p)->v;
}
template <class T, int N>
__device__ __forceinline__ void put(T* p, typename Vec<T, N>::V v) {
  reinterpret_cast<Loose<T, N>*>(p)->v = v;
}
// .. the first `there` of which exist.
template <class T, int N>
__device__ __forceinline__ typename Vec<T, N>::V get(const T* p, int there) {
  if (there >= N) return get<T, N>(p);
  typename Vec<T, N>::V v = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < there) v[i] = p[i];
  return v;
}
template <class T, int N>
__device__ __forceinline__ void put(T* p, int there, typename Vec<T, N>::V v) {
  if (there >= N) return put<T, N>(p, v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < there) p[i] = v[i];
}

// The codes of N values, four to a word.  Where neither the scale's reciprocal nor
// the remainders leave the ordinary numbers, the quotient comes from Markstein's
// theorem (IBM Journal of Research and Development 34, 1990): with the reciprocal y
// of s correctly rounded and q a faithful rounding of v / s, q + (v - q s) y rounds
// to the quotient correctly rounded.  v y is off by less than 1.5 steps, one such
// correction makes it faithful, the second exact.  Elsewhere the division decides.
// (bf16 rows hold exact borders of two codes in about every second thousand values,
// so that a quick answer that leaves those to the division is slower.)
struct Coder {
  float s, inv;
  bool quick;
  __device__ __forceinline__ explicit Coder(float scale)
      : s(scale), inv(__fdiv_rn(1.f, scale)), quick(scale >= 0x1p-90f && scale <= 0x1p100f) {}
  template <int N>
  __device__ __forceinline__ void codes(const float (&v)[N], uint32_t (&out)[N / 4]) const {
    if (quick) {
      constexpr float kMagic = 0x1.8p23f;  // added to a small number: its nearest integer in the low bits
      uint32_t b[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float q = v[i] * inv;
        q = __builtin_fmaf(__builtin_fmaf(-q, s, v[i]), inv, q);
        q = __builtin_fmaf(__builtin_fmaf(-q, s, v[i]), inv, q);
        b[i] = __float_as_uint(q + kMagic);
      }
#pragma unroll
      for (int i = 0; i < N; i += 4)
        out[i / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[i + 3], b[i + 2], 0x0C0C0400u),
                                           __builtin_amdgcn_perm(b[i + 1], b[i], 0x0C0C0400u), 0x05040100u);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4)
        out[i / 4] = (uint32_t)(code_of(v[i], s) & 255) | (uint32_t)(code_of(v[i + 1], s) & 255) << 8 |
                     (uint32_t)(code_of(v[i + 2], s) & 255) << 16 | (uint32_t)code_of(v[i + 3], s) << 24;
    }
  }
};

}  // namespace qmoe_i8
