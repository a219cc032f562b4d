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
//
// A row belongs to a wave, four waves or sixteen, whose threads keep it in
// registers between its passes (the sum of squares, the largest value, the
// codes); longer rows are read again for each.  Threads move 16 bytes at a time
// at whatever address a row begins.  Bound by HBM from some thousands of rows
// on (norm of 8192 x 2048 bf16 with the residual, its sum and the norm written:
// 28 us, 5.4 TB/s; 65536 x 2048 fp32 to codes: 114 us, 5.9
// TB/s; the values back: 58 us, 6.9 TB/s), by one chain of loads, two reductions and
// the stores below (one row of 2048: 2.6 us per call in a graph, quantised alone
// 2.2, its values 2.2).
#include "int8_codes.h"
#include "lanes.h"
#include "tiles.h"

namespace {

using namespace qmoe_i8;
// As put, past the caches: for what is written whole and read later, if at all.
// The values of 65536 x 2048 in bf16 take 58 us so and 71 without, in fp32 92 and
// 144; the norm of 4096 x 2048 with its residual's sum and itself 10.6 and 13.4.
// Not for codes, which a product reads next (quantisation and product of 16384
// rows: 163 us so, 157 without).
template <class T, int N>
__device__ __forceinline__ void put_nt(T* p, int there, typename Vec<T, N>::V v) {
  typedef typename Vec<T, N>::V At __attribute__((aligned(1)));
  if (there >= N) __builtin_nontemporal_store(v, reinterpret_cast<At*>(p));
  else put<T, N>(p, there, v);
}

// v combined over the TPR threads of a row (whole waves; the whole block from two waves on).
template <int TPR, class T, class Op>
__device__ __forceinline__ T over_row(T v, T* shared, Op op) {
  v = qmoe_lanes::over<64>(v, op);
  if constexpr (TPR > 64) {
    constexpr int kW = TPR / 64;
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int i = 1; i < kW; ++i) v = op(v, shared[i]);
  }
  return v;
}

// The rounding to the type in one instruction.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T rounded(float f) {
  if constexpr (DT == QMOE_BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  else return Elem<DT>::store(f);
}

struct RowArgs {
  const void* x;
  const void* r;  // the residual; null: none
  const void* w;  // the norm's weight, of the rows' type or fp32; null: ones
  int w_f32;
  int64_t rows, D;
  double eps;
  int8_t* q;
  float* s;
  void* sum;   // h; null: not written
  void* norm;  // v in the rows' type; null: not written
};

template <int DT>
constexpr int kVec = 16 / sizeof(typename Elem<DT>::T);

// TPR threads per row, blocks of at least 256; NV vectors of N elements per
// thread in registers, 0: rows of any length, read again.  A row's last vector
// ends with it: where N does not divide D it overlaps the one before, whose
// elements it has as well (they are counted once).  No load stands in a branch,
// so that all of a thread's are under way together.  D < N: one vector of which
// D elements exist (SHORT).
// With ids, the first block makes the table of their tiles: a launch less in front
// of a product of sorted rows (40,960 ids and 4096 x 2048 values 10.3 -> 8.1 us, 700
// and 93 x 1296 5.9 -> 3.8).
template <int DT, bool NORM, int TPR, int NV, bool SHORT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void int8_rows_kernel(RowArgs a, qmoe_tiles::Sorted table) {
  typedef typename Elem<DT>::T T;
  constexpr int N = kVec<DT>, kKept = NV ? NV : 1;
  typedef typename Vec<T, N>::V V;
  __shared__ double sums[TPR / 64];
  __shared__ uint32_t tops[TPR / 64];
  int64_t block = blockIdx.x;
  if constexpr (!NORM) {
    if (table.ids && block-- == 0) {
      constexpr int T = TPR < 256 ? 256 : TPR;
      __shared__ int lds[qmoe_tiles::kSamples];
      return qmoe_tiles::from_sorted<T>(table, lds);
    }
  }
  const int64_t row = TPR < 256 ? block * (256 / TPR) + threadIdx.x / TPR : block;
  if (row >= a.rows) return;
  const int lane = threadIdx.x % TPR, D = (int)a.D, there = SHORT ? D : N;
  const int64_t base = row * a.D;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* r = NORM && a.r ? static_cast<const T*>(a.r) + base : nullptr;
  const int64_t vecs = (a.D + N - 1) / N;
  const auto place = [&](int64_t i) { return SHORT ? 0 : (int)min(i * N, (int64_t)D - N); };
  // f(place in the registers, first element, element that the vector begins with as its own) for this thread's vectors
  const auto each = [&](auto f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) f(k, place(lane + k * TPR), (int64_t)(lane + k * TPR) * N);
    } else {
      for (int64_t i = lane; i < vecs; i += TPR) f(0, place(i), i * N);
    }
  };
  V xv[kKept], rv[kKept];
  const auto load = [&](int k, int c) {
    xv[k] = get<T, N>(x + c, there);
    if (NORM && r) rv[k] = get<T, N>(r + c, there);
  };
  float kept[kKept][N];
  const auto h = [&](int k, int c) {
    if (!NV) load(k, c);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      kept[k][i] = Elem<DT>::load(xv[k][i]);
      if (NORM && r) kept[k][i] = Elem<DT>::load(rounded<DT>(kept[k][i] + Elem<DT>::load(rv[k][i])));
    }
  };
  const auto narrow = [&](int k) {
    V o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = rounded<DT>(kept[k][i]);
    return o;
  };
  each([&](int k, int c, int64_t) {
    if (NV) load(k, c);
  });
  if constexpr (NV > 0) each([&](int k, int c, int64_t) { h(k, c); });
  float rstd = 1.f, lift = 1.f;
  if constexpr (NORM) {
    double ss = 0.0;
    each([&](int k, int c, int64_t own) {
      if (!NV) h(k, c);
      if (a.sum && own < a.D) put_nt<T, N>(static_cast<T*>(a.sum) + base + c, there, narrow(k));
      if (__any(own != c)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (c + i >= own && i < there) ss = fma((double)kept[k][i], (double)kept[k][i], ss);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fma((double)kept[k][i], (double)kept[k][i], ss);
      }
    });
    ss = over_row<TPR>(ss, sums, [](double p, double q) { return p + q; });
    const double r64 = 1.0 / sqrt(ss / (double)a.D + a.eps);
    // past fp32's range in rows near its ends: the row takes a part of the factor, a power of two
    if (r64 > 0x1p100) lift = 0x1p64f;
    else if (r64 < 0x1p-100) lift = 0x1p-64f;
    rstd = (float)(r64 / lift);
  }
  const auto normed = [&](int k, int c) {
    if constexpr (!NORM) return;
    if (lift != 1.f) {
#pragma unroll
      for (int i = 0; i < N; ++i) kept[k][i] *= lift;
    }
    if (!a.w) {
#pragma unroll
      for (int i = 0; i < N; ++i) kept[k][i] *= rstd;
    } else if (a.w_f32) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const typename Vec<float, 4>::V q = get<float, 4>(static_cast<const float*>(a.w) + c + i, there - i);
#pragma unroll
        for (int j = 0; j < 4; ++j) kept[k][i + j] = kept[k][i + j] * rstd * q[j];
      }
    } else {
      const V q = get<T, N>(static_cast<const T*>(a.w) + c, there);
#pragma unroll
      for (int i = 0; i < N; ++i) kept[k][i] = kept[k][i] * rstd * Elem<DT>::load(q[i]);
    }
  };
  uint32_t top = 0;
  each([&](int k, int c, int64_t) {
    if (!NV) h(k, c);
    normed(k, c);
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, i < there ? magnitude(kept[k][i]) : 0u);
  });
  top = over_row<TPR>(top, tops, [](uint32_t p, uint32_t q) { return max(p, q); });
  const float s = scale_of(top);
  if (lane == 0) a.s[row] = s;
  const Coder coder(s);
  each([&](int k, int c, int64_t own) {
    if (!NV) {
      h(k, c);
      normed(k, c);
    }
    uint32_t code[N / 4];
    coder.codes(kept[k], code);
    if (own >= a.D) return;
    if (NORM && a.norm) put_nt<T, N>(static_cast<T*>(a.norm) + base + c, there, narrow(k));
    put<uint8_t, N>(reinterpret_cast<uint8_t*>(a.q) + base + c, there, __builtin_bit_cast(typename Vec<uint8_t, N>::V, code));
  });
}

// Codes times their row's scale: TPR threads per row, 256 per block, NV vectors of a thread under way together.
template <int DT, int TPR, int NV>
__global__ __launch_bounds__(256) void int8_values_kernel(const int8_t* __restrict__ q, const float* __restrict__ s,
                                                          int64_t rows, int64_t D, typename Elem<DT>::T* __restrict__ out) {
  typedef typename Elem<DT>::T T;
  constexpr int N = kVec<DT>;
  typedef typename Vec<int8_t, N>::V C;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const int64_t base = row * D;
  const float sc = s[row];
  const int there = (int)min(D, (int64_t)N);
  const auto place = [&](int64_t own) { return D < N ? 0 : min(own, D - N); };  // the last vector ends with the row
  for (int64_t own = (threadIdx.x % TPR) * N; own < D; own += NV * TPR * N) {
    C v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = get<int8_t, N>(q + base + place(own + k * TPR * N), there);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (own + k * TPR * N >= D) break;
      typename Vec<T, N>::V o;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = rounded<DT>((float)v[k][i] * sc);
      put_nt<T, N>(out + base + place(own + k * TPR * N), there, o);
    }
  }
}

template <int DT, bool NORM, int TPR, int NV, bool SHORT = false>
void launch_form(const RowArgs& a, const qmoe_tiles::Sorted& table, hipStream_t st) {
  constexpr int kPer = TPR < 256 ? 256 / TPR : 1;
  int8_rows_kernel<DT, NORM, TPR, NV, SHORT><<<dim3((unsigned)((a.rows + kPer - 1) / kPer + (table.ids ? 1 : 0))), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(a, table);
}
// A wave per row where the rows alone fill the chip and a thread holds up to
// four vectors, else a vector per thread where that is possible: a thread's
// vectors cost 1 to 2 us each one after the other.  Norms of bf16 rows, wave /
// four waves per row (us): 1024 x 1000 5.1 / 5.9, 512 x 2048 6.9 / 5.0, 2048 x
// 2048 8.9 / 9.1, 4096 x 4096 (eight vectors a thread / two) 24.5 / 20.6 (measured
// with the norm's stores through the caches).
template <int DT, bool NORM>
void launch_type(const RowArgs& a, const qmoe_tiles::Sorted& table, hipStream_t st) {
  const int64_t vecs = (a.D + kVec<DT> - 1) / kVec<DT>;
  if (a.D < kVec<DT>) launch_form<DT, NORM, 64, 1, true>(a, table, st);
  else if (vecs <= 64) launch_form<DT, NORM, 64, 1>(a, table, st);
  else if (vecs <= 128 && a.rows >= 1024) launch_form<DT, NORM, 64, 2>(a, table, st);
  else if (vecs <= 256 && a.rows >= 2048) launch_form<DT, NORM, 64, 4>(a, table, st);
  else if (vecs <= 256) launch_form<DT, NORM, 256, 1>(a, table, st);
  else if (vecs <= 512) launch_form<DT, NORM, 256, 2>(a, table, st);
  else if (vecs <= 1024) launch_form<DT, NORM, 1024, 1>(a, table, st);
  else if (vecs <= 4096) launch_form<DT, NORM, 1024, 4>(a, table, st);
  else launch_form<DT, NORM, 1024, 0>(a, table, st);
}
template <bool NORM>
int launch_rows(const RowArgs& a, int dtype, const qmoe_tiles::Sorted& table, hipStream_t st) {
  if (dtype == QMOE_BF16) launch_type<QMOE_BF16, NORM>(a, table, st);
  else if (dtype == QMOE_FP16) launch_type<QMOE_FP16, NORM>(a, table, st);
  else launch_type<QMOE_FP32, NORM>(a, table, st);
  return qmoe::launch_status("int8_rows_kernel");
}
// A wave per row and four vectors a thread where the rows fill the chip (4096 x
// 2048: 4.5 us, by four waves 5.4 with stores through the caches), else threads enough for one or two each.
template <int DT>
void launch_values(const int8_t* q, const float* s, int64_t rows, int64_t D, void* out, hipStream_t st) {
  typedef typename Elem<DT>::T T;
  T* o = static_cast<T*>(out);
  const int64_t vecs = (D + kVec<DT> - 1) / kVec<DT>;
  const auto wave = dim3((unsigned)((rows + 3) / 4)), block = dim3((unsigned)rows);
  if (vecs <= 64) int8_values_kernel<DT, 64, 1><<<wave, dim3(256), 0, st>>>(q, s, rows, D, o);
  else if (vecs <= 256 && rows >= 2048) int8_values_kernel<DT, 64, 4><<<wave, dim3(256), 0, st>>>(q, s, rows, D, o);
  else if (vecs <= 256) int8_values_kernel<DT, 256, 1><<<block, dim3(256), 0, st>>>(q, s, rows, D, o);
  else if (vecs <= 512) int8_values_kernel<DT, 256, 2><<<block, dim3(256), 0, st>>>(q, s, rows, D, o);
  else int8_values_kernel<DT, 256, 4><<<block, dim3(256), 0, st>>>(q, s, rows, D, o);
}

constexpr int kThreads = 1024;  // of a block, at most

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
  return launch_rows<false>({x, nullptr, nullptr, 0, rows, K, 0.0, codes, scales, nullptr, nullptr}, dtype, {},
                            qmoe::as_stream(stream));
}

extern "C" int qmoe_int8_quantize_sorted(const void* x, int dtype, int64_t rows, int64_t K, int8_t* codes, float* scales,
                                         const int32_t* sorted_ids, int64_t n_rows, int32_t num_experts,
                                         int32_t tile_rows, int32_t* offsets, int32_t* tile_row, int32_t* tile_exp,
                                         int32_t* ntiles, int64_t max_tiles, void* stream) {
  bool run;
  const int rc = check_rows(rows, K, dtype, x, codes, scales, &run);
  if (rc != QMOE_OK) return rc;
  if (n_rows < 0 || num_experts <= 0 || tile_rows <= 0 || max_tiles < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (n_rows > 0x7FFFFFFF) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many rows");
  if (!offsets || !tile_row || !tile_exp || !ntiles || (n_rows && !sorted_ids)) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(x) || !qmoe::aligned16(codes)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "x and codes must be 16-byte aligned");
  if (!run || n_rows == 0) {  // a launch each
    const int rc2 = run ? qmoe_int8_quantize(x, dtype, rows, K, codes, scales, stream) : QMOE_OK;
    return rc2 != QMOE_OK ? rc2 : qmoe_build_tiles_clamped(sorted_ids, n_rows, num_experts, tile_rows, offsets, tile_row,
                                                           tile_exp, ntiles, max_tiles, stream);
  }
  return launch_rows<false>({x, nullptr, nullptr, 0, rows, K, 0.0, codes, scales, nullptr, nullptr}, dtype,
                            {sorted_ids, n_rows, num_experts, tile_rows, offsets, tile_row, tile_exp, ntiles, max_tiles, true},
                            qmoe::as_stream(stream));
}

extern "C" int qmoe_int8_dequantize(const int8_t* codes, const float* scales, int64_t rows, int64_t K, int dtype,
                                    void* out, void* stream) {
  bool run;
  const int rc = check_rows(rows, K, dtype, out, codes, scales, &run);
  if (rc != QMOE_OK || !run || K == 0) return rc;
  if (!qmoe::aligned16(out) || !qmoe::aligned16(codes)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "codes and out must be 16-byte aligned");
  hipStream_t st = qmoe::as_stream(stream);
  if (dtype == QMOE_BF16) launch_values<QMOE_BF16>(codes, scales, rows, K, out, st);
  else if (dtype == QMOE_FP16) launch_values<QMOE_FP16>(codes, scales, rows, K, out, st);
  else launch_values<QMOE_FP32>(codes, scales, rows, K, out, st);
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
  return launch_rows<true>({x, residual, weight, weight_dtype == QMOE_FP32, rows, D, eps, codes, scales, sum, norm}, dtype,
                           {}, qmoe::as_stream(stream));
}
