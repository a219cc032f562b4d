// Quantisation to and from mxfp4 (the format is in mxfp4.h).
//
// For a block of 32 with largest magnitude m, the scale is 2^e with
// e = floor(log2 m) - 2, clamped to [-127, 127] (OCP MX v1.0, 6.3: the largest
// power of two in m over the largest one in an element, 4 = 2^2); every
// element is x / 2^e rounded to the nearest e2m1 value, ties to the even code,
// magnitudes past 6 to 6 (v_cvt_scalef32_pk_fp4_*, which divides by the power
// of two exactly).  A block that holds a NaN or an infinity gets the scale
// byte 255, so all of it reads back as NaN.  An all-zero block keeps its signs
// under byte 0.
//
// Both directions are bound by HBM: 2 or 4 bytes an element on one side,
// 17/32 on the other.  134M fp32 values: 109 us (5.6 TB/s) and 83 us back.
#include "mxfp4.h"

namespace {

using namespace qmoe_mx;

typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2_t;

// Largest of v over each aligned group of four lanes (quad permutes).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
  return v;
}

// Eight consecutive elements as fp32 (exact for the 16-bit types).
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t u, float (&f)[8]) {
  if constexpr (DT == QMOE_FP32) {
    const f32x4_t a = __builtin_nontemporal_load(static_cast<const f32x4_t*>(x) + 2 * u);
    const f32x4_t b = __builtin_nontemporal_load(static_cast<const f32x4_t*>(x) + 2 * u + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  } else {
    const i32x4_t a = __builtin_nontemporal_load(static_cast<const i32x4_t*>(x) + u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t p = (uint32_t)a[i];  // a copy: a bit cast of a[i] itself reads a[0]
      if constexpr (DT == QMOE_BF16) {
        f[2 * i] = bf16lo(p);
        f[2 * i + 1] = bf16hi(p);
      } else {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, p);
        f[2 * i] = (float)h[0];
        f[2 * i + 1] = (float)h[1];
      }
    }
  }
}

// The scale byte of the block that four neighbouring lanes hold, eight elements
// each.
__device__ __forceinline__ uint32_t quad_scale(const float (&f)[8]) {
  // magnitudes compare as integers; an infinity or a NaN is past all finite ones
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  m = quad_max(m);
  // the exponent field of a normal m is floor(log2 m) + 127; a subnormal one
  // (field 0) and fields up to 2 clamp to byte 0, a non-finite one is 255
  const int field = (int)(m >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - 2, 0);
}
// The word of codes of eight elements under a scale byte.
__device__ __forceinline__ uint32_t quantize8(const float (&f)[8], uint32_t byte) {
  const float sc = scale_of(byte);
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[0], f[1], sc, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[2], f[3], sc, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[4], f[5], sc, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[6], f[7], sc, 3);
  return byte == 255u ? 0u : q;
}

// One thread per word of codes, four neighbouring lanes per block.
template <int DT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* __restrict__ x, int64_t words,
                                                          uint32_t* __restrict__ w, uint8_t* __restrict__ s) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= words) return;  // whole quads: words is a multiple of four
  float f[8];
  load8<DT>(x, u, f);
  const uint32_t byte = quad_scale(f);
  w[u] = quantize8(f, byte);
  if ((threadIdx.x & 3) == 0) s[u >> 2] = (uint8_t)byte;
}

// Quantises bf16 rows and lays their scales and the weights' out in lines: the
// first blocks take sixteen threads per row and group of 128 columns, each one
// word of codes; the others 64 weight rows each, a lane per row.  Bound by the
// weights' scales, a 17th of their bytes read and written.
__global__ __launch_bounds__(256) void mx_quantize_lines_kernel(const uint4* __restrict__ x, int64_t n_x, int64_t K,
                                                                uint32_t* __restrict__ xq, uint32_t* __restrict__ xl,
                                                                int64_t xblocks, const uint8_t* __restrict__ s,
                                                                int64_t rows, int64_t N, uint32_t* __restrict__ sl) {
  const int64_t G = (K + 127) / 128, units = K / kBlock;
  if ((int64_t)blockIdx.x < xblocks) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t line = u / 16;  // row * G + group
    const int l = (int)(u % 16);
    const int64_t row = min(line / G, n_x - 1), g = line % G;
    const int64_t word = g * 16 + l;  // of the row
    const bool in = line < n_x * G && word < K / 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (in) load8<QMOE_BF16>(x, row * (K / 8) + word, f);
    const uint32_t byte = in ? quad_scale(f) : 0u;
    if (in) xq[row * (K / 8) + word] = quantize8(f, byte);
    // lane 0 of sixteen collects the four blocks' bytes
    uint32_t four = byte;
#pragma unroll
    for (int b = 1; b < 4; ++b) four |= (uint32_t)__shfl_down((int)byte, 4 * b, 64) << (8 * b);
    if (l == 0 && line < n_x * G) xl[g * n_x + row] = four;
    return;
  }
  const int64_t r = ((int64_t)blockIdx.x - xblocks) * 64 + threadIdx.x % 64;
  if (r >= rows) return;
  const int64_t e = r / N, n = r - e * N;
  const uint8_t* src = s + r * units;
  uint32_t* dst = sl + e * G * N + n;
  const bool whole = units % 16 == 0 && (reinterpret_cast<uintptr_t>(s) & 15) == 0;
  for (int64_t g0 = threadIdx.x / 64 * 4; g0 < G; g0 += 16) {
    uint32_t v[4];
    if (whole) {
      const uint4 q = *reinterpret_cast<const uint4*>(src + 4 * g0);
      v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = 0;
        for (int b = 0; b < 4; ++b)
          if (4 * (g0 + i) + b < units) v[i] |= (uint32_t)src[4 * (g0 + i) + b] << (8 * b);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (g0 + i < G) dst[(g0 + i) * N] = v[i];
  }
}

// A thread makes 16 bytes of values at a time, so that a wave's stores are
// whole lines: a word's eight in 16 bits, or half a word's four in 32 (with a
// word's 32 bytes per thread a wave's stores left every other 16 bytes of each
// line to a second one: 134M values to fp32 in 217 us, now 83 us, 7.3 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* __restrict__ w,
                                                            const uint8_t* __restrict__ s, int64_t pieces,
                                                            i32x4_t* __restrict__ out) {
  constexpr int kPer = DT == QMOE_FP32 ? 2 : 1;  // pieces per word
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= pieces) return;
  uint32_t q = w[u / kPer];
  const float sc = scale_of(s[u / (4 * kPer)]);
  i32x4_t v;
  if constexpr (DT == QMOE_BF16) {
    uint32_t o[4];
    unpack8(q, sc, o);
    v = i32x4_t{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
  } else if constexpr (DT == QMOE_FP32) {
    if (u & 1) q >>= 16;
    const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 0);
    const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 1);
    v = __builtin_bit_cast(i32x4_t, f32x4_t{p0[0], p0[1], p1[0], p1[1]});
  } else {
    const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 0);
    const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 1);
    const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 2);
    const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 3);
    const f16x2_t h[4] = {{(_Float16)p0[0], (_Float16)p0[1]}, {(_Float16)p1[0], (_Float16)p1[1]},
                          {(_Float16)p2[0], (_Float16)p2[1]}, {(_Float16)p3[0], (_Float16)p3[1]}};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(int, h[i]);
  }
  __builtin_nontemporal_store(v, out + u);
}

// per: threads per word of codes
int check(const void* x, const void* w, const void* s, int dtype, int64_t rows, int64_t K, int per) {
  if (dtype != QMOE_BF16 && dtype != QMOE_FP16 && dtype != QMOE_FP32)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  if (rows < 0 || K < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes rows=%lld K=%lld", (long long)rows, (long long)K);
  if (K % kBlock) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: must be a multiple of 32", (long long)K);
  if (rows == 0 || K == 0) return QMOE_OK;
  if (!x || !w || !s) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(x) || !qmoe::aligned4(w))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "the values must be 16-byte aligned, the codes 4-byte aligned");
  if (rows > ((int64_t)0xFFFFFFFF - 255) / per / (K / 8)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many elements");
  return QMOE_OK;
}

}  // namespace

extern "C" int qmoe_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t K, uint32_t* w, uint8_t* scales,
                                   void* stream) {
  const int rc = check(x, w, scales, dtype, rows, K, 1);
  if (rc != QMOE_OK || rows == 0 || K == 0) return rc;
  const int64_t words = rows * (K / 8);
  const dim3 grid((unsigned)((words + 255) / 256)), block(256);
  hipStream_t st = qmoe::as_stream(stream);
  if (dtype == QMOE_BF16) mx_quantize_kernel<QMOE_BF16><<<grid, block, 0, st>>>(x, words, w, scales);
  else if (dtype == QMOE_FP16) mx_quantize_kernel<QMOE_FP16><<<grid, block, 0, st>>>(x, words, w, scales);
  else mx_quantize_kernel<QMOE_FP32><<<grid, block, 0, st>>>(x, words, w, scales);
  return qmoe::launch_status("mx_quantize_kernel");
}

extern "C" int qmoe_mxfp4_dequantize(const uint32_t* w, const uint8_t* scales, int64_t rows, int64_t K, int dtype,
                                     void* out, void* stream) {
  const int rc = check(out, w, scales, dtype, rows, K, dtype == QMOE_FP32 ? 2 : 1);
  if (rc != QMOE_OK || rows == 0 || K == 0) return rc;
  const int64_t pieces = rows * (K / 8) * (dtype == QMOE_FP32 ? 2 : 1);
  const dim3 grid((unsigned)((pieces + 255) / 256)), block(256);
  hipStream_t st = qmoe::as_stream(stream);
  i32x4_t* o = static_cast<i32x4_t*>(out);
  if (dtype == QMOE_BF16) mx_dequantize_kernel<QMOE_BF16><<<grid, block, 0, st>>>(w, scales, pieces, o);
  else if (dtype == QMOE_FP16) mx_dequantize_kernel<QMOE_FP16><<<grid, block, 0, st>>>(w, scales, pieces, o);
  else mx_dequantize_kernel<QMOE_FP32><<<grid, block, 0, st>>>(w, scales, pieces, o);
  return qmoe::launch_status("mx_dequantize_kernel");
}

extern "C" int qmoe_mxfp4_quantize_lines(const uint16_t* x, int64_t n_x, int64_t K, uint32_t* xq, const uint8_t* scales,
                                         int32_t num_experts, int64_t N, uint32_t* lines, int64_t line_words,
                                         void* stream) {
  const int rc = check(x, xq, scales, QMOE_BF16, n_x, K, 1);
  if (rc != QMOE_OK) return rc;
  if (num_experts < 0 || N < 0 || line_words < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (n_x == 0 || K == 0) return QMOE_OK;
  const int64_t G = (K + 127) / 128;
  if (N > 0x7FFFFFFF || K > 0x7FFFFFFF || num_experts * N > ((int64_t)1 << 40) / G || n_x > ((int64_t)1 << 40) / G)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  const int64_t rows = num_experts * N;
  if (!lines || !qmoe::aligned4(lines)) return qmoe::fail(QMOE_ERR_INVALID, "lines must be 4-byte aligned");
  if (line_words < (rows + n_x) * G) return qmoe::fail(QMOE_ERR_WORKSPACE, "lines hold %lld words, %lld are needed", (long long)line_words, (long long)((rows + n_x) * G));
  const int64_t xblocks = (n_x * G + 15) / 16, blocks = xblocks + (rows + 63) / 64;
  if (qmoe::too_many(blocks, 256)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  mx_quantize_lines_kernel<<<dim3((unsigned)blocks), dim3(256), 0, qmoe::as_stream(stream)>>>(
      reinterpret_cast<const uint4*>(x), n_x, K, xq, lines + rows * G, xblocks, scales, rows, N, lines);
  return qmoe::launch_status("mx_quantize_lines_kernel");
}
