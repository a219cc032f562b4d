// Products of 8-bit integers with few rows, each with an expert of its own
// (int8_product.h): matrix-vector kernels, the weights read straight from HBM.
//
// LPR lanes side by side cover one weight row, 16 codes of a load at a time,
// through v_dot4_i32_i8.
#include "int8_product.h"

namespace {

using namespace qmoe_i8;

constexpr int kWaves = 4;

// One wave: 64 / LPR groups of lanes, NR weight rows each, for one row of x.
template <int LPR, int NR>
__global__ __launch_bounds__(64 * kWaves) void int8_qmv_kernel(Product a) {
  constexpr int kRows = (64 / LPR) * NR;  // weight rows per wave
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int sub = lane / LPR, li = lane % LPR;
  const int64_t r = blockIdx.y;
  const int64_t n0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  if (n0 >= a.N) return;
  const int64_t e = a.experts ? min(max(a.experts[r], 0), a.num_experts - 1) : 0;
  const int64_t xr = x_row_of(a, r);
  const int units = (int)(a.K / 16);
  const i32x4_t* x = reinterpret_cast<const i32x4_t*>(a.x) + xr * units;
  const i32x4_t* w[NR];
  int acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t n = min(n0 + i * (64 / LPR) + sub, a.N - 1);  // rows past the end: the last again, not stored
    w[i] = reinterpret_cast<const i32x4_t*>(a.w) + (e * a.N + n) * units;
    acc[i] = 0;
  }
  for (int u = li; u < units; u += LPR) {
    i32x4_t q[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) q[i] = w[i][u];
    const i32x4_t xv = x[u];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i] = __builtin_amdgcn_sdot4(q[i][j], xv[j], acc[i], false);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    int v = acc[i];
#pragma unroll
    for (int m = LPR / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    const int64_t n = n0 + i * (64 / LPR) + sub;
    if (li == 0 && n < a.N) put(a, r * a.N + n, scaled(v, a.sx[xr], a.sw[e * a.N + n]));
  }
}

template <int LPR, int NR>
int launch(const Product& a, hipStream_t st) {
  constexpr int kRows = (64 / LPR) * NR * kWaves;
  const dim3 grid((unsigned)((a.N + kRows - 1) / kRows), (unsigned)a.n_rows);
  if (qmoe::too_many((int64_t)grid.x * grid.y, 64 * kWaves))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld: too many for weights of this size", (long long)a.n_rows);
  int8_qmv_kernel<LPR, NR><<<grid, dim3(64 * kWaves), 0, st>>>(a);
  return qmoe::launch_status("int8_qmv_kernel");
}

}  // namespace

int qmoe_i8::check(const Product& a, bool* run) {
  *run = false;
  if (a.n_rows < 0 || a.n_x < 0 || a.N < 0 || a.K < 0 || a.num_experts < 0 || a.x_div <= 0)
    return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (!qmoe::size_of(a.dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "out_dtype=%d", a.dtype);
  if (a.n_rows == 0 || a.N == 0) return QMOE_OK;
  if (a.n_x == 0 || a.num_experts == 0) return qmoe::fail(QMOE_ERR_INVALID, "no activation rows or no experts");
  if (a.K == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty contraction");
  if (!a.x || !a.sx || !a.w || !a.sw || !a.out) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (a.K % 16 || a.K > kMaxK)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: must be a multiple of 16, at most %lld", (long long)a.K, (long long)kMaxK);
  if (a.N > 0x7FFFFFFF || a.n_rows > 0x7FFFFFFF || a.n_x > 0x7FFFFFFF)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  if (!qmoe::aligned16(a.x) || !qmoe::aligned16(a.w) || !qmoe::aligned16(a.out))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "codes and out must be 16-byte aligned");
  *run = true;
  return QMOE_OK;
}

extern "C" int qmoe_int8_gather_qqmv(const int8_t* x, const float* sx, int64_t n_x, const int32_t* x_rows, int32_t x_div,
                                     const int32_t* experts, int64_t n_rows, const int8_t* w, const float* sw,
                                     int32_t num_experts, int64_t N, int64_t K, int out_dtype, void* out, void* stream) {
  Product a{x, sx, x_rows, n_rows, n_x, x_div, experts, w, sw, num_experts, N, K, nullptr, nullptr, nullptr, nullptr, out, out_dtype};
  bool run;
  const int rc = check(a, &run);
  if (rc != QMOE_OK || !run) return rc;
  if (n_rows > 65535) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld > 65535", (long long)n_rows);
  return launch<64, 2>(a, qmoe::as_stream(stream));
}
