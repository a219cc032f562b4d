// Microscaled 4-bit floating point (mxfp4) on gfx950: pieces shared by the
// kernels of mxfp4.hip, mxfp4_qmv.hip and mxfp4_gemm.hip.
//
// Format (OCP Microscaling Formats v1.0, MXFP4): blocks of 32 elements along
// the packed axis share a scale 2^(byte - 127) (byte 255: not a number); an
// element is a sign bit over one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (e2m1).  Eight
// codes to a 32-bit word, low bits first, so one block is one 16-byte unit.
//
// v_cvt_scalef32_pk_bf16_fp4 turns two codes into two bf16 values, scaled by
// the exponent field of an fp32 operand: byte << 23 is that operand for every
// byte (0 gives 2^-127, 255 gives NaN).  The product of an e2m1 value and a
// power of two has two significant bits, so the bf16 is exact, subnormals
// included, up to the largest finite bf16; 4 and 6 at 2^126, and 2 to 6 at
// 2^127, are infinite.
#pragma once

#include "common.h"

namespace qmoe_mx {

constexpr int kBlock = 32;  // elements per scale

// Scales in lines: per group of 128 columns a line of one word per row, the
// row's four scale bytes (0 past the last block), so that copies of
// consecutive rows' scales read consecutive words: word [e][g][n] of [experts]
// [ceil(K/128)][N], and after those of the weights [g][row] of the activations.

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// Byte b of four scale bytes as the conversions' operand, in one rotation: they
// use the exponent field alone, whatever the sign and the mantissa bits are.
__device__ __forceinline__ float scale_of(uint32_t four, int b) {
  return __uint_as_float(__builtin_amdgcn_alignbit(four, four, (8 * b + 9) & 31));
}

// Codes 2*SEL and 2*SEL + 1 of a word as a bf16 pair, low half first.
template <int SEL>
__device__ __forceinline__ uint32_t pair_of(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, SEL));
}
// The word's eight elements as four bf16 pairs.
__device__ __forceinline__ void unpack8(uint32_t word, float scale, uint32_t (&o)[4]) {
  o[0] = pair_of<0>(word, scale);
  o[1] = pair_of<1>(word, scale);
  o[2] = pair_of<2>(word, scale);
  o[3] = pair_of<3>(word, scale);
}

}  // namespace qmoe_mx
