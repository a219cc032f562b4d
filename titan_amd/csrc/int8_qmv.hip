// Products of 8-bit integers with few rows, each with an expert of its own
// (int8_product.h): matrix-vector kernels, the weights read straight from HBM.
//
// LPR lanes side by side cover one weight row, 16 codes of a load at a time,
// through v_dot4_i32_i8.  Rows that are no codes yet are quantised by every block
// for itself, the first weights on their way meanwhile: a launch less, and the
// same codes as int8_rows.hip's.  Bound by the latency of one dependent HBM round
// trip at one token (per call in a graph, 4096 x 2048: 4.6 us for 8.4 MB, from
// bf16 values 4.8; top-10 of 1024 x 2048 6.4 and 6.6), by HBM and the caches at
// more (six tokens 21).
#include "int8_codes.h"
#include "int8_product.h"
#include "lanes.h"

namespace {

using namespace qmoe_i8;

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int64_t kMaxValues = 16384;  // longest row that a block quantises, kept in LDS
constexpr int kCodes = 3;              // DT of rows that are codes

// The codes of a row of K values in LDS and their scale (16-byte units, K a multiple of 16).
template <int DT>
__device__ __forceinline__ float quantize_row(const void* x_, int64_t K, char* codes, uint32_t* tops) {
  typedef typename Elem<DT>::T T;
  constexpr int N = 16 / sizeof(T);
  typedef typename Vec<T, N>::V V;
  const V* x = static_cast<const V*>(x_);
  const int vecs = (int)(K / N);
  // a vector per thread stays in registers, more are read again
  V kept = x[min((int)threadIdx.x, vecs - 1)];
  uint32_t top = 0;
  const auto largest = [&](const V& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, magnitude(Elem<DT>::load(v[i])));
  };
  largest(kept);
  for (int i = threadIdx.x + kThreads; i < vecs; i += kThreads) largest(x[i]);
  top = qmoe_lanes::over<64>(top, [](uint32_t p, uint32_t q) { return max(p, q); });
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = max(top, tops[i]);
  const float s = scale_of(top);
  const Coder coder(s);
  for (int base = 0; base < vecs; base += kThreads) {  // all lanes: the coder's waves decide together
    const int i = base + threadIdx.x;
    if (base) kept = x[min(i, vecs - 1)];
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = Elem<DT>::load(kept[j]);
    uint32_t c[N / 4];
    coder.codes(v, c);
    if (i < vecs) {
      if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(c[0], c[1]);
      else *reinterpret_cast<uint32_t*>(codes + i * 4) = c[0];
    }
  }
  __syncthreads();
  return s;
}

// One wave: 64 / LPR groups of lanes, NR weight rows each, for one row of x.
template <int DT, int LPR, int NR>
__global__ __launch_bounds__(kThreads) void int8_qmv_kernel(Product a) {
  constexpr int kRows = (64 / LPR) * NR;  // weight rows per wave
  constexpr bool kValues = DT != kCodes;
  __shared__ __attribute__((aligned(16))) char codes[kValues ? kMaxValues : 16];
  __shared__ uint32_t tops[kWaves];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int sub = lane / LPR, li = lane % LPR;
  const int64_t r = blockIdx.y;
  const int64_t n0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  const int64_t e = a.experts ? min(max(a.experts[r], 0), a.num_experts - 1) : 0;
  const int64_t xr = x_row_of(a, r);
  const int units = (int)(a.K / 16);
  const i32x4_t* w[NR];
  int acc[NR];
  i32x4_t q[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t n = min(n0 + i * (64 / LPR) + sub, a.N - 1);  // rows past the end: the last again, not stored
    w[i] = reinterpret_cast<const i32x4_t*>(a.w) + (e * a.N + n) * units;
    acc[i] = 0;
    q[i] = w[i][min(li, units - 1)];
  }
  float sx;
  const i32x4_t* x;
  if constexpr (kValues) {
    sx = quantize_row<DT>(static_cast<const typename Elem<DT>::T*>(static_cast<const void*>(a.x)) + xr * a.K, a.K, codes, tops);
    x = reinterpret_cast<const i32x4_t*>(codes);
  } else {
    sx = a.sx[xr];
    x = reinterpret_cast<const i32x4_t*>(a.x) + xr * units;
  }
  for (int u = li; u < units; u += LPR) {
    const i32x4_t xv = x[u];
    i32x4_t next[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) next[i] = w[i][min(u + LPR, units - 1)];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i] = __builtin_amdgcn_sdot4(q[i][j], xv[j], acc[i], false);
      q[i] = next[i];
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int v = qmoe_lanes::over<LPR>(acc[i], [](int p, int s) { return p + s; });
    const int64_t n = n0 + i * (64 / LPR) + sub;
    if (li == 0 && n < a.N) put(a, r * a.N + n, scaled(v, sx, a.sw[e * a.N + n]));
  }
}

template <int DT, int LPR, int NR>
int launch(const Product& a, hipStream_t st) {
  constexpr int kRows = (64 / LPR) * NR * kWaves;
  // in eights, so that the rows of x that take the same weights run on the same XCD (block ids are dealt round-robin) and
  // find them in its L2 (eight rows by 4099 of 2080: 15.4 -> 9.8 us); what is past the end works on the last weight row
  const int64_t blocks = (a.N + kRows - 1) / kRows;
  const dim3 grid((unsigned)(a.n_rows > 1 ? (blocks + 7) / 8 * 8 : blocks), (unsigned)a.n_rows);
  if (qmoe::too_many((int64_t)grid.x * grid.y, kThreads))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld: too many for weights of this size", (long long)a.n_rows);
  int8_qmv_kernel<DT, LPR, NR><<<grid, dim3(kThreads), 0, st>>>(a);
  return qmoe::launch_status("int8_qmv_kernel");
}
// Lanes per weight row: as many as leave each two loads one after the other,
// and where the rows are many about four of them, in fewer and longer waves.  64 /
// 32 / 16 lanes, codes (us per call in a graph): 4096 rows of 2048 4.6 / 5.1 / 7.2,
// 16384 6.1 / 5.7 / 7.5; 4096 rows of 1024 (8 experts) 3.3 / 2.9 / 3.8, 24576 5.9 /
// 4.8 / 4.6; 20480 rows of 2048 (two tokens x top-10) 10.7 / 9.5 / 9.9.  Values, eight
// rows by 4096: of 1040 6.1 / 6.1 / 5.3, of 2064 11.9 / 8.2 / 9.1, of 3008 12.7 / 9.5 / 11.2.
template <int DT>
int launch_lanes(const Product& a, hipStream_t st) {
  const bool many = a.n_rows * a.N >= 16384;
  const int64_t loads = many ? 4 : 2, lanes = (a.K / 16 + loads - 1) / loads, spare = many ? 3 : 2;  // halves
  if (lanes > 16 * spare) return launch<DT, 64, 2>(a, st);
  return lanes > 8 * spare ? launch<DT, 32, 2>(a, st) : launch<DT, 16, 2>(a, st);
}

}  // namespace

int qmoe_i8::check(const Product& a, bool values, bool* run) {
  *run = false;
  if (a.n_rows < 0 || a.n_x < 0 || a.N < 0 || a.K < 0 || a.num_experts < 0 || a.x_div <= 0)
    return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (!qmoe::size_of(a.dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "out_dtype=%d", a.dtype);
  if (a.n_rows == 0 || a.N == 0) return QMOE_OK;
  if (a.n_x == 0 || a.num_experts == 0) return qmoe::fail(QMOE_ERR_INVALID, "no activation rows or no experts");
  if (a.K == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty contraction");
  if (!a.x || (!a.sx && !values) || !a.w || !a.sw || !a.out) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (a.K % 16 || a.K > kMaxK)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: must be a multiple of 16, at most %lld", (long long)a.K, (long long)kMaxK);
  if (a.N > 0x7FFFFFFF || a.n_rows > 0x7FFFFFFF || a.n_x > 0x7FFFFFFF)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  if (!qmoe::aligned16(a.x) || !qmoe::aligned16(a.w) || !qmoe::aligned16(a.out))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "x, w and out must be 16-byte aligned");
  *run = true;
  return QMOE_OK;
}

extern "C" int qmoe_int8_gather_qqmv(const int8_t* x, const float* sx, int64_t n_x, const int32_t* x_rows, int32_t x_div,
                                     const int32_t* experts, int64_t n_rows, const int8_t* w, const float* sw,
                                     int32_t num_experts, int64_t N, int64_t K, int out_dtype, void* out, void* stream) {
  Product a{x, sx, x_rows, n_rows, n_x, x_div, experts, w, sw, num_experts, N, K, nullptr, nullptr, nullptr, nullptr, out, out_dtype};
  bool run;
  const int rc = check(a, false, &run);
  if (rc != QMOE_OK || !run) return rc;
  if (n_rows > 65535) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld > 65535", (long long)n_rows);
  return launch_lanes<kCodes>(a, qmoe::as_stream(stream));
}

extern "C" int qmoe_int8_gather_qmv(const void* x, int dtype, int64_t n_x, const int32_t* x_rows, int32_t x_div,
                                    const int32_t* experts, int64_t n_rows, const int8_t* w, const float* sw,
                                    int32_t num_experts, int64_t N, int64_t K, int out_dtype, void* out, void* stream) {
  Product a{static_cast<const int8_t*>(x), nullptr, x_rows, n_rows, n_x, x_div, experts, w, sw, num_experts, N, K,
            nullptr, nullptr, nullptr, nullptr, out, out_dtype};
  if (!qmoe::size_of(dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  bool run;
  const int rc = check(a, true, &run);
  if (rc != QMOE_OK || !run) return rc;
  if (n_rows > 65535) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_rows=%lld > 65535", (long long)n_rows);
  if (K > kMaxValues) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: rows of values have at most %lld", (long long)K, (long long)kMaxValues);
  hipStream_t st = qmoe::as_stream(stream);
  if (dtype == QMOE_BF16) return launch_lanes<QMOE_BF16>(a, st);
  return dtype == QMOE_FP16 ? launch_lanes<QMOE_FP16>(a, st) : launch_lanes<QMOE_FP32>(a, st);
}
