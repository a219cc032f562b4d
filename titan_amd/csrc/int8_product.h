// What the kernels of products of 8-bit integers share (format in int8_rows.hip).
//
//   out[r, n] = (sum_k x[r, k] w[n, k]) * sx[r] * sw[n]
//
// Sums are exact in 32 bits up to kMaxK (codes of -128 included); the scales
// are applied in fp32 and the result is rounded once.
#pragma once

#include "elem.h"

namespace qmoe_i8 {

constexpr int64_t kMaxK = 131056;  // the last multiple of 16 below 2^31 / 2^14

struct Product {
  const int8_t* x;        // [n_x, K]
  const float* sx;        // [n_x]
  const int32_t* x_rows;  // null: row r reads activation row r / x_div
  int64_t n_rows, n_x;    // output rows; activation rows
  int32_t x_div;
  const int32_t* experts;  // the few-rows kernel's expert of each row; null: expert 0
  const int8_t* w;         // [E, N, K]
  const float* sw;         // [E, N]
  int32_t num_experts;
  int64_t N, K;
  const int32_t *offsets, *tile_row, *tile_exp, *ntiles;  // all null: one expert, rows in order
  void* out;
  int dtype;
};

__device__ __forceinline__ int64_t x_row_of(const Product& a, int64_t r) {
  const int64_t t = a.x_rows ? (int64_t)a.x_rows[r] : r / a.x_div;
  return min(max(t, (int64_t)0), a.n_x - 1);
}

// A sum times both scales: the row's first where it is of ordinary size, so
// that the product with it neither overflows nor underflows, else the smaller
// one first, whose product overflows only where the result does and loses
// nothing to underflow that the result keeps.
__device__ __forceinline__ bool ordinary(float sx) {
  const float v = fabsf(sx);
  return (v >= 0x1p-60f && v <= 0x1p60f) || v == 0.f;
}
__device__ __forceinline__ float scaled(int acc, float sx, float sw) {
  const bool first = ordinary(sx) || fabsf(sx) < fabsf(sw);
  return (float)acc * (first ? sx : sw) * (first ? sw : sx);
}
__device__ __forceinline__ void put(const Product& a, int64_t i, float v) {
  if (a.dtype == QMOE_FP32) static_cast<float*>(a.out)[i] = v;
  else if (a.dtype == QMOE_FP16) static_cast<_Float16*>(a.out)[i] = (_Float16)v;
  else static_cast<uint16_t*>(a.out)[i] = (uint16_t)f32_to_bf16(v);
}

// Argument checks of the entry points; QMOE_OK with *run = false: nothing to do.
// values: x has no scales yet.
int check(const Product& a, bool values, bool* run);

}  // namespace qmoe_i8
