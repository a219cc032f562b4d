// Rows in 8 bits with one fp32 scale each, the values back, and the RMS norm
// that leaves its result in that form.
//
//   scale   s = max |v| / 127                     (fp32, correctly rounded)
//   code    q = rint(v / s) in [-127, 127]         (a row of zeros: 0, 0)
//   norm    h = T(x + r),  v = h / sqrt(mean(h^2) + eps) * w
//
// A row that holds a NaN or an infinity has the scale NaN and codes 0, so that
// it reads back as NaN throughout and spoils no other row.  The squares are
// summed in 64 bits: no value of the types overflows or vanishes there.
#include "elem.h"

namespace {

constexpr int kThreads = 256;

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

struct RowArgs {
  const void* x;
  const void* r;  // the residual; null: none
  const void* w;  // the norm's weight, of the rows' type or fp32; null: ones
  int w_f32;
  int64_t D;
  double eps;
  int8_t* q;
  float* s;
  void* sum;   // h; null: not written
  void* norm;  // v in the rows' type; null: not written
};

// One block per row.
template <int DT, bool NORM>
__global__ __launch_bounds__(kThreads) void int8_rows_kernel(RowArgs a) {
  typedef typename Elem<DT>::T T;
  __shared__ double sums[kThreads / 64];
  __shared__ uint32_t tops[kThreads / 64];
  const int64_t row = blockIdx.x, base = row * a.D;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* r = a.r ? static_cast<const T*>(a.r) + base : nullptr;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const auto h_of = [&](int64_t c) {
    const float v = Elem<DT>::load(x[c]);
    return r ? Elem<DT>::load(Elem<DT>::store(v + Elem<DT>::load(r[c]))) : v;
  };
  float rstd = 1.f;
  if constexpr (NORM) {
    double ss = 0.0;
    for (int64_t c = threadIdx.x; c < a.D; c += kThreads) {
      const float h = h_of(c);
      if (a.sum) static_cast<T*>(a.sum)[base + c] = Elem<DT>::store(h);
      ss = fma((double)h, (double)h, ss);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
    if (lane == 0) sums[wave] = ss;
    __syncthreads();
    ss = sums[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) ss += sums[i];
    rstd = (float)(1.0 / sqrt(ss / (double)a.D + a.eps));
  }
  const auto v_of = [&](int64_t c) {
    float v = h_of(c);
    if constexpr (NORM) {
      v *= rstd;
      if (a.w) v *= a.w_f32 ? static_cast<const float*>(a.w)[c] : Elem<DT>::load(static_cast<const T*>(a.w)[c]);
    }
    return v;
  };
  uint32_t top = 0;
  for (int64_t c = threadIdx.x; c < a.D; c += kThreads) top = max(top, magnitude(v_of(c)));
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) top = max(top, tops[i]);
  const float s = scale_of(top);
  if (threadIdx.x == 0) a.s[row] = s;
  for (int64_t c = threadIdx.x; c < a.D; c += kThreads) {
    const float v = v_of(c);
    a.q[base + c] = (int8_t)code_of(v, s);
    if (NORM && a.norm) static_cast<T*>(a.norm)[base + c] = Elem<DT>::store(v);
  }
}

// One block per row: codes times the row's scale.
template <int DT>
__global__ __launch_bounds__(kThreads) void int8_values_kernel(const int8_t* __restrict__ q, const float* __restrict__ s,
                                                               int64_t D, typename Elem<DT>::T* __restrict__ out) {
  const int64_t base = (int64_t)blockIdx.x * D;
  const float sc = s[blockIdx.x];
  for (int64_t c = threadIdx.x; c < D; c += kThreads) out[base + c] = Elem<DT>::store((float)q[base + c] * sc);
}

template <bool NORM>
int launch_rows(const RowArgs& a, int64_t rows, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)rows), block(kThreads);
  if (dtype == QMOE_BF16) int8_rows_kernel<QMOE_BF16, NORM><<<grid, block, 0, st>>>(a);
  else if (dtype == QMOE_FP16) int8_rows_kernel<QMOE_FP16, NORM><<<grid, block, 0, st>>>(a);
  else int8_rows_kernel<QMOE_FP32, NORM><<<grid, block, 0, st>>>(a);
  return qmoe::launch_status("int8_rows_kernel");
}

// QMOE_OK with *run = false: nothing to do.
int check_rows(int64_t rows, int64_t D, int dtype, const void* in, const int8_t* q, const float* s, bool* run) {
  *run = false;
  if (!qmoe::size_of(dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  if (rows < 0 || D < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (rows == 0) return QMOE_OK;
  if (!s || (D && (!in || !q))) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (D > 0x7FFFFFFF || qmoe::too_many(rows, kThreads))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "%lld rows of %lld: too large", (long long)rows, (long long)D);
  *run = true;
  return QMOE_OK;
}

}  // namespace

extern "C" int qmoe_int8_quantize(const void* x, int dtype, int64_t rows, int64_t K, int8_t* codes, float* scales,
                                  void* stream) {
  bool run;
  const int rc = check_rows(rows, K, dtype, x, codes, scales, &run);
  if (rc != QMOE_OK || !run) return rc;
  if (!qmoe::aligned16(x) || !qmoe::aligned16(codes)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "x and codes must be 16-byte aligned");
  return launch_rows<false>({x, nullptr, nullptr, 0, K, 0.0, codes, scales, nullptr, nullptr}, rows, dtype,
                            qmoe::as_stream(stream));
}

extern "C" int qmoe_int8_dequantize(const int8_t* codes, const float* scales, int64_t rows, int64_t K, int dtype,
                                    void* out, void* stream) {
  bool run;
  const int rc = check_rows(rows, K, dtype, out, codes, scales, &run);
  if (rc != QMOE_OK || !run || K == 0) return rc;
  if (!qmoe::aligned16(out) || !qmoe::aligned16(codes)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "codes and out must be 16-byte aligned");
  hipStream_t st = qmoe::as_stream(stream);
  const dim3 grid((unsigned)rows), block(kThreads);
  if (dtype == QMOE_BF16) int8_values_kernel<QMOE_BF16><<<grid, block, 0, st>>>(codes, scales, K, static_cast<uint16_t*>(out));
  else if (dtype == QMOE_FP16) int8_values_kernel<QMOE_FP16><<<grid, block, 0, st>>>(codes, scales, K, static_cast<_Float16*>(out));
  else int8_values_kernel<QMOE_FP32><<<grid, block, 0, st>>>(codes, scales, K, static_cast<float*>(out));
  return qmoe::launch_status("int8_values_kernel");
}

extern "C" int qmoe_int8_rms_norm(const void* x, const void* residual, const void* weight, int weight_dtype, int dtype,
                                  int64_t rows, int64_t D, double eps, int8_t* codes, float* scales, void* sum,
                                  void* norm, void* stream) {
  bool run;
  const int rc = check_rows(rows, D, dtype, x, codes, scales, &run);
  if (rc != QMOE_OK) return rc;
  if (!(eps >= 0.0) || eps > 1e30) return qmoe::fail(QMOE_ERR_INVALID, "eps=%g", eps);
  if (weight && weight_dtype != dtype && weight_dtype != QMOE_FP32)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "weight_dtype=%d: the rows' type or fp32", weight_dtype);
  if (!run) return QMOE_OK;
  if (D == 0) return qmoe::fail(QMOE_ERR_INVALID, "rows without elements have no norm");
  for (const void* p : {x, residual, weight, (const void*)codes, (const void*)sum, (const void*)norm})
    if (!qmoe::aligned16(p)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "the rows and the weight must be 16-byte aligned");
  return launch_rows<true>({x, residual, weight, weight_dtype == QMOE_FP32, D, eps, codes, scales, sum, norm}, rows,
                           dtype, qmoe::as_stream(stream));
}
