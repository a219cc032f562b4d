// Products of mxfp4 weights with few rows of bf16 activations: matrix-vector
// kernels, the weights of each row read straight from HBM (format in mxfp4.h).
//
// Forward, out[r, n] = sum_k x[r, k] W[e_r, n, k]: a lane's 16-byte load of
// codes is exactly one block of 32, so it needs one scale byte, and LPR lanes
// side by side cover one weight row.  Codes become bf16 pairs by the scaled
// conversion (exact) and go through v_dot2_f32_bf16 with the activation's
// pairs: 32 instructions per 32 codes.  Bound by the latency of one dependent
// HBM round trip at one token (per call in a graph, 4096 x 2048: 4.0 us for 4.5
// MB; top-10 of 1024 x 2048: 5.7 us for 11 MB), by the caches and HBM at more
// (six tokens 16.2 us).
//
// Transposed, out[r, k] = sum_n x[r, n] W[e_r, n, k]: a lane owns the 32
// outputs of one block column and walks n, four rows' loads ahead; sixteen
// lanes and sixteen waves share the n of one block of 128 outputs and add up
// their sums, through LDS and in a fixed order.
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
constexpr int kTUnits = 4;               // block columns (of 32 outputs) per workgroup
constexpr int kTOut = kTUnits * kBlock;  // outputs per workgroup
constexpr int kTRows = 64 / kTUnits;     // rows n a wave takes at once
constexpr int kTAhead = 4;               // of which so many batches are in flight

__global__ __launch_bounds__(64 * kTWaves) void mx_qmv_t_kernel(QmvArgs a) {
  __shared__ float part[kTWaves][kTOut];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = lane / kTRows, sub = lane % kTRows;  // block column, row n
  const int64_t r = blockIdx.y;
  const int64_t e = expert_of(a, r);
  const uint16_t* x = a.x + x_row_of(a, r) * a.ldx;
  const int units = (int)(a.K / kBlock);
  const int64_t u = min((int64_t)blockIdx.x * kTUnits + c, (int64_t)units - 1);  // past the end: not stored
  const uint4* w = reinterpret_cast<const uint4*>(a.w) + e * a.N * units + u;
  const uint8_t* s = a.s + e * a.N * units + u;
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
  constexpr int kStep = kTWaves * kTRows;
  for (int64_t n0 = wave * kTRows + sub; n0 < a.N; n0 += kTAhead * kStep) {
    uint4 q[kTAhead];
    float sc[kTAhead], xv[kTAhead];
#pragma unroll
    for (int i = 0; i < kTAhead; ++i) {
      const int64_t n = n0 + i * kStep;
      const bool in = n < a.N;
      const int64_t at = in ? n * units : 0;
      q[i] = w[at];
      sc[i] = scale_of(in ? s[at] : 0u);  // past the end: 0 times what is there, which is finite
      xv[i] = in ? bf16_to_f32(x[n]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kTAhead; ++i) {
      const uint32_t qw[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t p[4];
        unpack8(qw[j], sc[i], p);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          acc[8 * j + 2 * t] = __builtin_fmaf(xv[i], bf16lo(p[t]), acc[8 * j + 2 * t]);
          acc[8 * j + 2 * t + 1] = __builtin_fmaf(xv[i], bf16hi(p[t]), acc[8 * j + 2 * t + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float v = group_sum<kTRows>(acc[i]);
    if (sub == 0) part[wave][c * kBlock + i] = v;
  }
  __syncthreads();
  if (threadIdx.x < kTOut) {
    const int64_t k = (int64_t)blockIdx.x * kTOut + threadIdx.x;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < kTWaves; ++j) v += part[j][threadIdx.x];
    if (k < a.K) put(a, r * a.K + k, v);
  }
}

int too_large(int64_t blocks, int64_t n_rows, int threads) {
  if (!qmoe::too_many(blocks * n_rows, threads)) return QMOE_OK;
  return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld: too many for weights of this size", (long long)n_rows);
}

template <int LPR, int NR>
int launch_fwd(const QmvArgs& a, hipStream_t st) {
  constexpr int kRows = (64 / LPR) * NR * kWaves;
  const int64_t blocks = (a.N + kRows - 1) / kRows;
  const int rc = too_large(blocks, a.n_rows, 64 * kWaves);
  if (rc != QMOE_OK) return rc;
  mx_qmv_kernel<LPR, NR><<<dim3((unsigned)blocks, (unsigned)a.n_rows), dim3(64 * kWaves), 0, st>>>(a);
  return qmoe::launch_status("mx_qmv_kernel");
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
    const int rc = too_large(grid.x, n_rows, 64 * kTWaves);
    if (rc != QMOE_OK) return rc;
    mx_qmv_t_kernel<<<grid, dim3(64 * kTWaves), 0, st>>>(a);
    return qmoe::launch_status("mx_qmv_t_kernel");
  }
  const int64_t units = K / kBlock;
  // Lanes per weight row: as many as give the fewest dependent passes (against
  // the fewest idle lanes, 16 or 32, one row of N = 4096: K = 2080 4.4 / 5.3 us, 1056 3.3 /
  // 3.4, 1536 3.4 / 4.1, 3200 4.8 / 7.1).
  const int lpr = units > 32 ? 64 : units > 16 ? 32 : 16;
  // Weight rows per wave: two, so that a row or a few fill the chip; four where
  // the pairs do (one token x top-10 of 1024 x 2048 5.7 / 6.1 us, two 8.9 / 8.2,
  // six 18.9 / 16.2).
  const bool many = n_rows >= 16;
  if (lpr == 64) return many ? launch_fwd<64, 4>(a, st) : launch_fwd<64, 2>(a, st);
  if (lpr == 32) return many ? launch_fwd<32, 4>(a, st) : launch_fwd<32, 2>(a, st);
  return many ? launch_fwd<16, 4>(a, st) : launch_fwd<16, 2>(a, st);
}
