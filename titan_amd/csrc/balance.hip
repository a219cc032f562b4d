// The router's balance loss with its gradient, and the experts' counts.
//
//   p_te = softmax of token t's logits          (fp32; a row of -inf: zeros)
//   c_e  = pairs of unmasked tokens routed to e, n unmasked tokens, k pairs a token
//   f_e  = c_e / (n k),  P_e = sum_t p_te / n    (t unmasked)
//   L    = E sum_e f_e P_e                       (n = 0: 0)
//   dL/dlogit_te = g E / n p_te (f_e - sum_e' f_e' p_te')   (t masked: exactly 0)
//
// The counts are constants of the gradient.  Sums over tokens go by blocks in
// a fixed order, nothing is added in floating point atomically, so results
// repeat bit for bit.
#include "elem.h"

namespace {

constexpr int kMaxE = 1024;
constexpr int kWaves = 4;
constexpr int kPer = kMaxE / 64;  // columns per lane
constexpr int kFinal = 1024;      // threads of the block that finishes

struct Tokens {
  const void* logits;
  const void* ids;      // int32 or int64 [T, k]
  const uint8_t* mask;  // null: every token counts
  int ids64;
  int64_t T;
  int E, k;
};

__device__ __forceinline__ bool live_of(const Tokens& a, int64_t t) { return !a.mask || a.mask[t]; }

// exp(x - max) of a row's columns lane, lane + 64, ..; returns 1 / their sum, 0 for a row of -inf.
template <int DT>
__device__ __forceinline__ float row_softmax(const Tokens& a, int64_t t, int lane, float (&p)[kPer]) {
  typedef typename Elem<DT>::T T;
  const T* x = static_cast<const T*>(a.logits) + t * a.E;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = lane + 64 * j;
    p[j] = c < a.E ? Elem<DT>::load(x[c]) : -INFINITY;
    top = fmaxf(top, p[j]);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    p[j] = lane + 64 * j < a.E ? __expf(p[j] - top) : 0.f;
    sum += p[j];
  }
  sum = group_sum<64>(sum);
  return sum == 0.f ? 0.f : 1.f / sum;
}

template <int DT>
__global__ __launch_bounds__(64 * kWaves) void balance_sums_kernel(Tokens a, float* __restrict__ psum,
                                                                   int32_t* __restrict__ csum,
                                                                   int32_t* __restrict__ nsum) {
  __shared__ int counts[kMaxE];
  __shared__ float part[kWaves][kMaxE];
  __shared__ int tokens;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (int c = threadIdx.x; c < a.E; c += 64 * kWaves) counts[c] = 0;
  if (threadIdx.x == 0) tokens = 0;
  __syncthreads();
  float acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < a.T; t += (int64_t)gridDim.x * kWaves) {
    if (!live_of(a, t)) continue;
    float p[kPer];
    const float inv = row_softmax<DT>(a, t, lane, p);
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] += p[j] * inv;
    for (int j = lane; j < a.k; j += 64) {
      const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[t * a.k + j] : static_cast<const int32_t*>(a.ids)[t * a.k + j];
      atomicAdd(&counts[min(max(id, (int64_t)0), (int64_t)a.E - 1)], 1);
    }
    if (lane == 0) atomicAdd(&tokens, 1);
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (lane + 64 * j < a.E) part[wave][lane + 64 * j] = acc[j];
  __syncthreads();
  for (int c = threadIdx.x; c < a.E; c += 64 * kWaves) {
    float v = part[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w][c];
    psum[(int64_t)blockIdx.x * a.E + c] = v;
    csum[(int64_t)blockIdx.x * a.E + c] = counts[c];
  }
  if (threadIdx.x == 0) nsum[blockIdx.x] = tokens;
}

// One block: the blocks' sums, and the loss and the counts of them.
__global__ __launch_bounds__(kFinal) void balance_loss_kernel(int E, int k, int blocks, const float* __restrict__ psum,
                                                              const int32_t* __restrict__ csum,
                                                              const int32_t* __restrict__ nsum,
                                                              int32_t* __restrict__ counts, float* __restrict__ loss,
                                                              int32_t* __restrict__ n_out) {
  __shared__ double sums[kFinal];
  const int c = threadIdx.x;
  int n = 0;
  for (int b = 0; b < blocks; ++b) n += nsum[b];
  double v = 0.0;
  if (c < E) {
    double p = 0.0;
    int64_t count = 0;
    for (int b = 0; b < blocks; ++b) {
      p += psum[(int64_t)b * E + c];
      count += csum[(int64_t)b * E + c];
    }
    counts[c] = (int32_t)count;
    v = p * (double)count;
  }
  sums[c] = v;
  __syncthreads();
  for (int m = kFinal / 2; m >= 1; m >>= 1) {
    if (c < m) sums[c] += sums[c + m];
    __syncthreads();
  }
  if (c == 0) {
    *loss = n ? (float)(sums[0] * E / ((double)n * n * k)) : 0.f;
    *n_out = n;
  }
}

template <int DT>
__global__ __launch_bounds__(64 * kWaves) void balance_grad_kernel(Tokens a, const int32_t* __restrict__ counts,
                                                                   const int32_t* __restrict__ n_,
                                                                   const float* __restrict__ g,
                                                                   void* __restrict__ out_) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t t = (int64_t)blockIdx.x * kWaves + wave;
  if (t >= a.T) return;
  T* out = static_cast<T*>(out_) + t * a.E;
  if (!live_of(a, t)) {
    for (int c = lane; c < a.E; c += 64) out[c] = Elem<DT>::store(0.f);
    return;
  }
  const float n = (float)n_[0];
  float p[kPer], f[kPer];
  const float inv = row_softmax<DT>(a, t, lane, p);
  float dot = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = lane + 64 * j;
    f[j] = c < a.E ? (float)counts[c] / (n * (float)a.k) : 0.f;
    p[j] *= inv;
    dot = __builtin_fmaf(f[j], p[j], dot);
  }
  dot = group_sum<64>(dot);
  const float scale = *g * (float)a.E / n;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = lane + 64 * j;
    if (c < a.E) out[c] = Elem<DT>::store(scale * (p[j] * (f[j] - dot)));
  }
}

// Blocks of the sums.
int64_t blocks_of(int64_t T) {
  const int64_t b = (T + 4 * kWaves - 1) / (4 * kWaves);
  return b < 1 ? 1 : b > 256 ? 256 : b;
}

int check(const Tokens& a, int64_t E, int64_t k, int dtype, bool ids) {
  if (!qmoe::size_of(dtype)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dtype=%d", dtype);
  if (a.T < 0 || E < 1 || k < 1) return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (E > kMaxE) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "E=%lld: at most %d experts", (long long)E, kMaxE);
  if (a.T > 0x7FFFFFFF / k) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many pairs");
  if (a.T && (!a.logits || (ids && !a.ids))) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(a.logits)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "logits must be 16-byte aligned");
  return QMOE_OK;
}

}  // namespace

extern "C" size_t qmoe_router_balance_workspace_size(int64_t T, int64_t E) {
  if (T < 0 || E < 1 || E > kMaxE) return 0;
  return (size_t)blocks_of(T) * (2 * E + 1) * 4;
}

extern "C" int qmoe_router_balance(const void* logits, int dtype, int64_t T, int64_t E, const void* ids, int ids64,
                                   int64_t k, const uint8_t* mask, float* loss, int32_t* counts, int32_t* n,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const Tokens a{logits, ids, mask, ids64, T, (int)E, (int)k};
  const int rc = check(a, E, k, dtype, true);
  if (rc != QMOE_OK) return rc;
  if (!loss || !counts || !n) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!workspace || workspace_bytes < qmoe_router_balance_workspace_size(T, E))
    return qmoe::fail(QMOE_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", workspace_bytes,
                      qmoe_router_balance_workspace_size(T, E));
  const int blocks = (int)blocks_of(T);
  float* psum = static_cast<float*>(workspace);
  int32_t* csum = reinterpret_cast<int32_t*>(psum + (size_t)blocks * E);
  int32_t* nsum = csum + (size_t)blocks * E;
  hipStream_t st = qmoe::as_stream(stream);
  const dim3 grid(blocks), block(64 * kWaves);
  if (dtype == QMOE_BF16) balance_sums_kernel<QMOE_BF16><<<grid, block, 0, st>>>(a, psum, csum, nsum);
  else if (dtype == QMOE_FP16) balance_sums_kernel<QMOE_FP16><<<grid, block, 0, st>>>(a, psum, csum, nsum);
  else balance_sums_kernel<QMOE_FP32><<<grid, block, 0, st>>>(a, psum, csum, nsum);
  if (const int rc2 = qmoe::launch_status("balance_sums_kernel")) return rc2;
  balance_loss_kernel<<<dim3(1), dim3(kFinal), 0, st>>>(a.E, a.k, blocks, psum, csum, nsum, counts, loss, n);
  return qmoe::launch_status("balance_loss_kernel");
}

extern "C" int qmoe_router_balance_grad(const void* logits, int dtype, int64_t T, int64_t E, int64_t k,
                                        const uint8_t* mask, const int32_t* counts, const int32_t* n, const float* dloss,
                                        void* dlogits, void* stream) {
  const Tokens a{logits, nullptr, mask, 0, T, (int)E, (int)k};
  const int rc = check(a, E, k, dtype, false);
  if (rc != QMOE_OK || T == 0) return rc;
  if (!counts || !n || !dloss || !dlogits) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (!qmoe::aligned16(dlogits)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "dlogits must be 16-byte aligned");
  const int64_t blocks = (T + kWaves - 1) / kWaves;
  if (qmoe::too_many(blocks, 64 * kWaves)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many tokens");
  hipStream_t st = qmoe::as_stream(stream);
  const dim3 grid((unsigned)blocks), block(64 * kWaves);
  if (dtype == QMOE_BF16) balance_grad_kernel<QMOE_BF16><<<grid, block, 0, st>>>(a, counts, n, dloss, dlogits);
  else if (dtype == QMOE_FP16) balance_grad_kernel<QMOE_FP16><<<grid, block, 0, st>>>(a, counts, n, dloss, dlogits);
  else balance_grad_kernel<QMOE_FP32><<<grid, block, 0, st>>>(a, counts, n, dloss, dlogits);
  return qmoe::launch_status("balance_grad_kernel");
}
