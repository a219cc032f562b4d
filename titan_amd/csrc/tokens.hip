// Tokens sorted by expert and back, with the scores applied, and the gradients
// of both.  Pair p = t * k + j is slot j of token t, inv[p] its sorted row, a
// permutation of the pairs (qmoe_route).
//
//   sort              xs[inv[t k + j]] = x[t]
//   its gradient      dx[t] = sum_j dxs[inv[t k + j]]
//   back              y[t]  = sum_j s[t, j] xs[inv[t k + j]]
//   its gradients     dxs[inv[p]] = s[p] dy[t],  ds[p] = <dy[t], xs[inv[p]]>
//
// Sums run in fp32 in slot order, whatever the rows' type, and are rounded
// once; nothing is added atomically, so results do not depend on timing.
// All of it is bound by memory: every row is read once and written once, and
// work goes by token, so that x[t] and dy[t] are read once for its k rows.  4096
// tokens x top-10 of 2048 bf16: the sort 34 us (5.4 TB/s; one wave per sorted
// row, which reads x[t] k times, 44), each sum 33 us (5.6 TB/s), both gradients
// of the way back 75 us (4.7 TB/s).
//
// A thread takes 16 bytes of a row where the row length is a multiple of 16
// bytes, one element otherwise (VEC).
#include "common.h"

namespace {

template <int DT>
struct Elem;
template <>
struct Elem<QMOE_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float load(T v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ T store(float f) { return (T)f32_to_bf16(f); }
};
template <>
struct Elem<QMOE_FP16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float load(T v) { return (float)v; }
  static __device__ __forceinline__ T store(float f) { return (_Float16)f; }
};
template <>
struct Elem<QMOE_FP32> {
  typedef float T;
  static __device__ __forceinline__ float load(T v) { return v; }
  static __device__ __forceinline__ T store(float f) { return f; }
};

// N consecutive elements, moved as one access of N * sizeof(T) bytes.
template <typename T, int N>
struct Vec {
  typedef T V __attribute__((ext_vector_type(N)));
};
template <typename T>
struct Vec<T, 1> {
  typedef T V;
};
template <typename T, int N>
__device__ __forceinline__ T at(const typename Vec<T, N>::V& v, int i) {
  if constexpr (N == 1) return v;
  else return v[i];
}
template <typename T, int N>
__device__ __forceinline__ void set(typename Vec<T, N>::V& v, int i, T x) {
  if constexpr (N == 1) v = x;
  else v[i] = x;
}

constexpr int kBatch = 8;  // rows in flight per thread

// One block per token, whose row is read once and written to its k places.
template <typename U>
__global__ __launch_bounds__(256) void sort_rows_kernel(const U* __restrict__ x, const int32_t* __restrict__ inv,
                                                        int64_t n, int k, int64_t units, U* __restrict__ out) {
  const int64_t t = blockIdx.x;
  for (int64_t c = threadIdx.x; c < units; c += blockDim.x) {
    const U v = x[t * units + c];
    for (int j = 0; j < k; ++j) {
      const int64_t i = min(max((int64_t)inv[t * k + j], (int64_t)0), n - 1);
      __builtin_nontemporal_store(v, out + i * units + c);
    }
  }
}

// y[t] = sum of the rows of token t's pairs, weighted by `scores` if given.
// With `first` the pairs of output row t are first[t] .. first[t + 1] - 1
// instead of t k .. t k + k - 1.
template <int IN, int OUT, int N>
__global__ __launch_bounds__(256) void unsort_sum_kernel(const void* __restrict__ xs_, int64_t n,
                                                         const int32_t* __restrict__ inv,
                                                         const float* __restrict__ scores,
                                                         const int32_t* __restrict__ first, int k, int64_t units,
                                                         void* __restrict__ y_) {
  typedef typename Elem<IN>::T TI;
  typedef typename Elem<OUT>::T TO;
  typedef typename Vec<TI, N>::V VI;
  typedef typename Vec<TO, N>::V VO;
  const VI* xs = static_cast<const VI*>(xs_);
  const int64_t c = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
  const int64_t t = blockIdx.x;
  if (c >= units) return;
  const int64_t p0 = first ? max(first[t], 0) : t * k;
  const int64_t p1 = first ? min((int64_t)first[t + 1], n) : p0 + k;
  float acc[N];
#pragma unroll
  for (int v = 0; v < N; ++v) acc[v] = 0.f;
  for (int64_t p = p0; p < p1; p += kBatch) {
    VI q[kBatch];
    float sc[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (p + b >= p1) break;
      const int64_t i = inv ? min(max((int64_t)inv[p + b], (int64_t)0), n - 1) : p + b;
      q[b] = __builtin_nontemporal_load(xs + i * units + c);
      sc[b] = scores ? scores[p + b] : 1.f;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (p + b >= p1) break;
#pragma unroll
      for (int v = 0; v < N; ++v) acc[v] = __builtin_fmaf(sc[b], Elem<IN>::load(at<TI, N>(q[b], v)), acc[v]);
    }
  }
  VO o;
#pragma unroll
  for (int v = 0; v < N; ++v) set<TO, N>(o, v, Elem<OUT>::store(acc[v]));
  __builtin_nontemporal_store(o, static_cast<VO*>(y_) + t * units + c);
}

// One block per token, its pairs in batches of kBatch: dxs of the batch's rows
// and their dot products with dy[t], summed over the block in a fixed order.
template <int DT, int N>
__global__ __launch_bounds__(256) void unsort_grad_kernel(const void* __restrict__ dy_, const void* __restrict__ xs_,
                                                          int64_t n, const int32_t* __restrict__ inv,
                                                          const float* __restrict__ scores, int k, int64_t units,
                                                          void* __restrict__ dxs_, float* __restrict__ ds) {
  typedef typename Elem<DT>::T T;
  typedef typename Vec<T, N>::V V;
  __shared__ float part[4][kBatch];
  const V* dy = static_cast<const V*>(dy_);
  const V* xs = static_cast<const V*>(xs_);
  V* dxs = static_cast<V*>(dxs_);
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
  for (int j0 = 0; j0 < k; j0 += kBatch) {
    int64_t row[kBatch];
    float sc[kBatch], dot[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t p = t * k + min(j0 + b, k - 1);
      row[b] = min(max((int64_t)inv[p], (int64_t)0), n - 1);
      sc[b] = scores[p];
      dot[b] = 0.f;
    }
    for (int64_t c = threadIdx.x; c < units; c += blockDim.x) {
      const V g = dy[t * units + c];
      V q[kBatch];
      if (ds) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (j0 + b >= k) break;
          q[b] = __builtin_nontemporal_load(xs + row[b] * units + c);
        }
      }
      if (dxs) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (j0 + b >= k) break;
          V o;
#pragma unroll
          for (int v = 0; v < N; ++v) set<T, N>(o, v, Elem<DT>::store(sc[b] * Elem<DT>::load(at<T, N>(g, v))));
          __builtin_nontemporal_store(o, dxs + row[b] * units + c);
        }
      }
      if (ds) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (j0 + b >= k) break;
#pragma unroll
          for (int v = 0; v < N; ++v)
            dot[b] = __builtin_fmaf(Elem<DT>::load(at<T, N>(g, v)), Elem<DT>::load(at<T, N>(q[b], v)), dot[b]);
        }
      }
    }
    if (!ds) continue;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const float v = group_sum<64>(dot[b]);
      if (lane == 0) part[wave][b] = v;
    }
    __syncthreads();
    if ((int)threadIdx.x < kBatch && j0 + (int)threadIdx.x < k) {
      float v = 0.f;
      for (int w = 0; w < waves; ++w) v += part[w][threadIdx.x];
      ds[t * k + j0 + threadIdx.x] = v;
    }
    __syncthreads();
  }
}

int size_of(int dtype) { return dtype == QMOE_FP32 ? 4 : dtype == QMOE_BF16 || dtype == QMOE_FP16 ? 2 : 0; }

// Threads for `units` work items along a row: whole waves, one at least, at most 256.
unsigned row_threads(int64_t units) { return (unsigned)(units >= 256 ? 256 : units <= 64 ? 64 : (units + 63) / 64 * 64); }
int too_large(int64_t blocks, unsigned threads) {
  if (!qmoe::too_many(blocks, threads)) return QMOE_OK;
  return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many rows of this length");
}

template <int IN, int OUT>
int launch_sum(const void* xs, int64_t n, const int32_t* inv, const float* scores, const int32_t* first, int64_t T,
               int k, int64_t D, void* y, hipStream_t st) {
  constexpr int N = 16 / sizeof(typename Elem<IN>::T);
  const bool vec = D % N == 0 && D * (int64_t)sizeof(typename Elem<OUT>::T) % 8 == 0;
  const int64_t units = vec ? D / N : D;
  const unsigned threads = row_threads(units);
  const int64_t cols = (units + threads - 1) / threads;
  if (cols > 65535) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "D=%lld too large", (long long)D);
  const dim3 grid((unsigned)T, (unsigned)cols);
  if (const int rc = too_large(T * cols, threads)) return rc;
  if (vec) unsort_sum_kernel<IN, OUT, N><<<grid, dim3(threads), 0, st>>>(xs, n, inv, scores, first, k, units, y);
  else unsort_sum_kernel<IN, OUT, 1><<<grid, dim3(threads), 0, st>>>(xs, n, inv, scores, first, k, units, y);
  return qmoe::launch_status("unsort_sum_kernel");
}

template <int DT>
int launch_grad(const void* dy, const void* xs, int64_t n, const int32_t* inv, const float* scores, int64_t T, int k,
                int64_t D, void* dxs, float* ds, hipStream_t st) {
  constexpr int N = 16 / sizeof(typename Elem<DT>::T);
  const bool vec = D % N == 0;
  const int64_t units = vec ? D / N : D;
  const dim3 grid((unsigned)T), block(row_threads(units));
  if (const int rc = too_large(T, block.x)) return rc;
  if (vec) unsort_grad_kernel<DT, N><<<grid, block, 0, st>>>(dy, xs, n, inv, scores, k, units, dxs, ds);
  else unsort_grad_kernel<DT, 1><<<grid, block, 0, st>>>(dy, xs, n, inv, scores, k, units, dxs, ds);
  return qmoe::launch_status("unsort_grad_kernel");
}

}  // namespace

extern "C" int qmoe_sort_rows(const void* x, int64_t T, const int32_t* inv, int64_t top_k, int64_t D, int dtype,
                              void* out, void* stream) {
  const int size = size_of(dtype);
  if (!size) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  if (T < 0 || top_k < 0 || D < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (T == 0 || top_k == 0 || D == 0) return QMOE_OK;
  if (!x || !inv || !out) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(x) || !qmoe::aligned16(out)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "rows must be 16-byte aligned");
  if (T > 0x7FFFFFFF / top_k) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many pairs");
  const int64_t n = T * top_k, bytes = D * size;
  const int unit = bytes % 16 == 0 ? 16 : size;
  const int64_t units = bytes / unit;
  const dim3 grid((unsigned)T), block(row_threads(units));
  if (const int rc = too_large(T, block.x)) return rc;
  hipStream_t st = qmoe::as_stream(stream);
  const int k = (int)top_k;
  if (unit == 16)
    sort_rows_kernel<<<grid, block, 0, st>>>(static_cast<const i32x4_t*>(x), inv, n, k, units, static_cast<i32x4_t*>(out));
  else if (unit == 4)
    sort_rows_kernel<<<grid, block, 0, st>>>(static_cast<const uint32_t*>(x), inv, n, k, units, static_cast<uint32_t*>(out));
  else
    sort_rows_kernel<<<grid, block, 0, st>>>(static_cast<const uint16_t*>(x), inv, n, k, units, static_cast<uint16_t*>(out));
  return qmoe::launch_status("sort_rows_kernel");
}

extern "C" int qmoe_unsort_sum(const void* xs, int64_t n, int dtype, const int32_t* inv, const float* scores,
                               const int32_t* first, int64_t T, int64_t top_k, int64_t D, int out_dtype, void* y,
                               void* stream) {
  if (!size_of(dtype) || (out_dtype != dtype && !(dtype == QMOE_FP32 && out_dtype == QMOE_BF16)))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d, out_dtype=%d", dtype, out_dtype);
  if (T < 0 || n < 0 || top_k < 0 || D < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (T == 0 || D == 0) return QMOE_OK;
  if (!y || (n && !xs)) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (top_k > 0x7FFFFFFF || n > 0x7FFFFFFF || T > 0x7FFFFFFE) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many pairs");
  if (!first && T * top_k != n) return qmoe::fail(QMOE_ERR_INVALID, "xs holds %lld rows, the pairs are %lld", (long long)n, (long long)(T * top_k));
  if (!qmoe::aligned16(xs) || !qmoe::aligned16(y)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "rows must be 16-byte aligned");
  hipStream_t st = qmoe::as_stream(stream);
  const int k = (int)top_k;
  if (dtype == QMOE_BF16) return launch_sum<QMOE_BF16, QMOE_BF16>(xs, n, inv, scores, first, T, k, D, y, st);
  if (dtype == QMOE_FP16) return launch_sum<QMOE_FP16, QMOE_FP16>(xs, n, inv, scores, first, T, k, D, y, st);
  if (out_dtype == QMOE_BF16) return launch_sum<QMOE_FP32, QMOE_BF16>(xs, n, inv, scores, first, T, k, D, y, st);
  return launch_sum<QMOE_FP32, QMOE_FP32>(xs, n, inv, scores, first, T, k, D, y, st);
}

extern "C" int qmoe_unsort_grad(const void* dy, const void* xs, int64_t n, int dtype, const int32_t* inv,
                                const float* scores, int64_t T, int64_t top_k, int64_t D, void* dxs, float* dscores,
                                void* stream) {
  if (!size_of(dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  if (T < 0 || n < 0 || top_k < 0 || D < 0) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (top_k > 0x7FFFFFFF || n > 0x7FFFFFFF || T > 0x7FFFFFFF) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many pairs");
  if (T * top_k != n) return qmoe::fail(QMOE_ERR_INVALID, "xs holds %lld rows, the pairs are %lld", (long long)n, (long long)(T * top_k));
  if (n == 0 || (!dxs && !dscores)) return QMOE_OK;
  if (D == 0 && !dscores) return QMOE_OK;
  if (!inv || !scores || (D && (!dy || (dscores && !xs)))) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(dy) || !qmoe::aligned16(xs) || !qmoe::aligned16(dxs))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "rows must be 16-byte aligned");
  hipStream_t st = qmoe::as_stream(stream);
  const int k = (int)top_k;
  if (dtype == QMOE_BF16) return launch_grad<QMOE_BF16>(dy, xs, n, inv, scores, T, k, D, dxs, dscores, st);
  if (dtype == QMOE_FP16) return launch_grad<QMOE_FP16>(dy, xs, n, inv, scores, T, k, D, dxs, dscores, st);
  return launch_grad<QMOE_FP32>(dy, xs, n, inv, scores, T, k, D, dxs, dscores, st);
}
