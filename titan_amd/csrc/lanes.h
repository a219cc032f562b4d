// Values combined across the lanes of a wave without LDS: DPP moves within a
// row of sixteen lanes, then swaps of rows and of halves (a ds_bpermute, which
// __shfl_xor becomes, costs a trip through the LDS crossbar per step).
#pragma once

#include "common.h"

namespace qmoe_lanes {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

// v (4 or 8 bytes) combined over aligned groups of L lanes, the same in all of
// them.  op is commutative.  L = 4, 8, 16, 32 or 64.
template <int L, class T, class Op>
__device__ __forceinline__ T over(T v, Op op) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    uint32_t w[W];
  };
  const auto step = [&](auto move) {
    const Words a = __builtin_bit_cast(Words, v);
    Words b;
#pragma unroll
    for (int i = 0; i < W; ++i) b.w[i] = move(a.w[i]);
    v = op(v, __builtin_bit_cast(T, b));
  };
  const auto swap = [&](auto pair) {  // pair gives both rows' (halves') values to both
    const Words a = __builtin_bit_cast(Words, v);
    Words b, c;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const auto p = pair(a.w[i]);
      b.w[i] = p[0], c.w[i] = p[1];
    }
    v = op(__builtin_bit_cast(T, b), __builtin_bit_cast(T, c));
  };
  step([](uint32_t x) { return dpp<0xB1>(x); });  // quad_perm 1,0,3,2
  step([](uint32_t x) { return dpp<0x4E>(x); });  // quad_perm 2,3,0,1
  if constexpr (L >= 8) step([](uint32_t x) { return dpp<0x141>(x); });   // row_half_mirror
  if constexpr (L >= 16) step([](uint32_t x) { return dpp<0x128>(x); });  // row_ror:8
  if constexpr (L >= 32) swap([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  if constexpr (L >= 64) swap([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}

}  // namespace qmoe_lanes
