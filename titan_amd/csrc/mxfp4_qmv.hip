// Products of mxfp4 weights with few rows of bf16 activations: matrix-vector
// kernels, the weights of each row read straight from HBM (format in mxfp4.h).
//
// Forward, out[r, n] = sum_k x[r, k] W[e_r, n, k]: a lane's 16-byte load of
// codes is exactly one block of 32, so it needs one scale byte, and LPR lanes
// side by side cover one weight row.  Codes become bf16 pairs by the scaled
// conversion (exact) and go through v_dot2_f32_bf16 with the activation's
// pairs: 32 instructions per 32 codes.  Bound by the latency of one dependent
// HBM round trip at one token, by HBM at more.
//
// Transposed, out[r, k] = sum_n x[r, n] W[e_r, n, k]: a lane owns the 32
// outputs of one block column and walks n; sixteen waves share the n of one
// block of 512 outputs and add up their sums through LDS in a fixed order.
#include "mxfp4.h"

namespace {

using namespace qmoe_mx;

constexpr int kWaves = 4;

struct QmvArgs {
  const uint16_t* x;
  const int32_t* x_rows;   // null: row i reads activation row i / x_div
  const int32_t* experts;  // null: expert 0
  int64_t n_rows, n_x;     // output rows; activation rows
  int32_t x_div;
  int64_t ldx;             // elements between activation rows
  const uint32_t* w;
  const uint8_t* s;
  int32_t num_experts;
  int64_t N, K;
  void* out;
  int out_f32;
};

__device__ __forceinline__ int64_t x_row_of(const QmvArgs& a, int64_t r) {
  const int64_t t = a.x_rows ? (int64_t)a.x_rows[r] : r / a.x_div;
  return min(max(t, (int64_t)0), a.n_x - 1);
}
__device__ __forceinline__ int64_t expert_of(const QmvArgs& a, int64_t r) {
  return a.experts ? min(max(a.experts[r], 0), a.num_experts - 1) : 0;
}
__device__ __forceinline__ void put(const QmvArgs& a, int64_t i, float v) {
  if (a.out_f32) static_cast<float*>(a.out)[i] = v;
  else static_cast<uint16_t*>(a.out)[i] = (uint16_t)f32_to_bf16(v);
}

// One wave: 64 / LPR groups of lanes, NR weight rows each, for one row of x.
template <int LPR, int NR>
__global__ __launch_bounds__(64 * kWaves) void mx_qmv_kernel(QmvArgs a) {
  constexpr int kRows = (64 / LPR) * NR;  // weight rows per wave
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int sub = lane / LPR, li = lane % LPR;
  const int64_t r = blockIdx.y;
  const int64_t n0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  if (n0 >= a.N) return;
  const int64_t e = expert_of(a, r);
  const uint4* x = reinterpret_cast<const uint4*>(a.x + x_row_of(a, r) * a.ldx);
  const int units = (int)(a.K / kBlock);
  const uint4* w[NR];
  const uint8_t* s[NR];
  float acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t n = min(n0 + i * (64 / LPR) + sub, a.N - 1);  // rows past the end: the last again, not stored
    w[i] = reinterpret_cast<const uint4*>(a.w) + (e * a.N + n) * units;
    s[i] = a.s + (e * a.N + n) * units;
    acc[i] = 0.f;
  }
  for (int u = li; u < units; u += LPR) {
    uint4 q[NR];
    uint32_t sb[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) q[i] = w[i][u], sb[i] = s[i][u];
    uint4 xv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = x[4 * u + i];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float sc = scale_of(sb[i]);
      const uint32_t qw[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t p[4];
        unpack8(qw[j], sc, p);
        acc[i] = dot2_bf16(p[0], xv[j].x, acc[i]);
        acc[i] = dot2_bf16(p[1], xv[j].y, acc[i]);
        acc[i] = dot2_bf16(p[2], xv[j].z, acc[i]);
        acc[i] = dot2_bf16(p[3], xv[j].w, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const float v = group_sum<LPR>(acc[i]);
    const int64_t n = n0 + i * (64 / LPR) + sub;
    if (li == 0 && n < a.N) put(a, r * a.N + n, v);
  }
}

constexpr int kTWaves = 16;
constexpr int kTUnits = 16;              // block columns (of 32 outputs) per workgroup
constexpr int kTOut = kTUnits * kBlock;  // outputs per workgroup

__global__ __launch_bounds__(64 * kTWaves) void mx_qmv_t_kernel(QmvArgs a) {
  __shared__ float part[kTWaves][kTOut];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = lane % kTUnits, sub = lane / kTUnits;  // block column, one of four rows n
  const int64_t r = blockIdx.y;
  const int64_t e = expert_of(a, r);
  const uint16_t* x = a.x + x_row_of(a, r) * a.ldx;
  const int units = (int)(a.K / kBlock);
  const int64_t u = (int64_t)blockIdx.x * kTUnits + c;
  const bool in = u < units;
  const uint4* w = reinterpret_cast<const uint4*>(a.w) + e * a.N * units + (in ? u : 0);
  const uint8_t* s = a.s + e * a.N * units + (in ? u : 0);
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
  for (int64_t n = wave * 4 + sub; n < a.N; n += 4 * kTWaves) {
    const uint4 q = w[n * units];
    const float sc = scale_of(s[n * units]);
    const float xv = bf16_to_f32(x[n]);
    const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t p[4];
      unpack8(qw[j], sc, p);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[8 * j + 2 * t] = __builtin_fmaf(xv, bf16lo(p[t]), acc[8 * j + 2 * t]);
        acc[8 * j + 2 * t + 1] = __builtin_fmaf(xv, bf16hi(p[t]), acc[8 * j + 2 * t + 1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    acc[i] += __shfl_xor(acc[i], 16);
    acc[i] += __shfl_xor(acc[i], 32);
  }
  if (sub == 0) {
#pragma unroll
    for (int i = 0; i < 32; ++i) part[wave][i * kTUnits + c] = acc[i];  // [element][column]: consecutive lanes, banks
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTOut; i += blockDim.x) {
    const int col = i / kBlock, el = i % kBlock;
    const int64_t k = (int64_t)blockIdx.x * kTOut + i;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < kTWaves; ++j) v += part[j][el * kTUnits + col];
    if (k < a.K) put(a, r * a.K + k, v);
  }
}

template <int LPR>
void launch_fwd(const QmvArgs& a, hipStream_t st) {
  constexpr int NR = 2;
  constexpr int kRows = (64 / LPR) * NR * kWaves;
  const dim3 grid((unsigned)((a.N + kRows - 1) / kRows), (unsigned)a.n_rows);
  mx_qmv_kernel<LPR, NR><<<grid, dim3(64 * kWaves), 0, st>>>(a);
}

}  // namespace

extern "C" int qmoe_mxfp4_gather_qmv(const uint16_t* x, int64_t n_x, int64_t ldx, const int32_t* x_rows, int32_t x_div,
                                     const int32_t* experts, int64_t n_rows, const uint32_t* w, const uint8_t* scales,
                                     int32_t num_experts, int64_t N, int64_t K, int transpose, int out_dtype,
                                     void* out, void* stream) {
  if (n_rows < 0 || n_x < 0 || N < 0 || K < 0 || num_experts < 0 || x_div <= 0 || ldx < (transpose ? K : N))
    return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (out_dtype != QMOE_BF16 && out_dtype != QMOE_FP32)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "out_dtype=%d", out_dtype);
  if (K % kBlock) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: must be a multiple of 32", (long long)K);
  const int64_t outs = transpose ? N : K;
  if (n_rows == 0 || outs == 0) return QMOE_OK;
  if ((transpose ? K : N) == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty contraction");
  if (n_x == 0 || num_experts == 0) return qmoe::fail(QMOE_ERR_INVALID, "no activation rows or no experts");
  if (!x || !w || !scales || !out) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(w) || (transpose && (!qmoe::aligned16(x) || ldx % 8)))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "codes and activation rows must be 16-byte aligned");
  if (n_rows > 65535 || N > 0x7FFFFFFF || K > 0x7FFFFFFF)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld > 65535, or sizes too large", (long long)n_rows);
  QmvArgs a{x, x_rows, experts, n_rows, n_x, x_div, ldx, w, scales, num_experts, N, K, out, out_dtype == QMOE_FP32};
  hipStream_t st = qmoe::as_stream(stream);
  if (!transpose) {
    const dim3 grid((unsigned)((K + kTOut - 1) / kTOut), (unsigned)n_rows);
    mx_qmv_t_kernel<<<grid, dim3(64 * kTWaves), 0, st>>>(a);
    return qmoe::launch_status("mx_qmv_t_kernel");
  }
  const int64_t units = K / kBlock;
  const auto slots = [&](int lpr) { return (units + lpr - 1) / lpr * lpr; };
  // lanes per weight row: as many as there are units, fewer where that wastes less of the last pass
  int lpr = 64;
  if (slots(32) < slots(lpr)) lpr = 32;
  if (slots(16) < slots(lpr)) lpr = 16;
  if (lpr == 64) launch_fwd<64>(a, st);
  else if (lpr == 32) launch_fwd<32>(a, st);
  else launch_fwd<16>(a, st);
  return qmoe::launch_status("mx_qmv_kernel");
}
