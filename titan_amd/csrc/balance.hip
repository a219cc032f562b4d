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
//
// L lanes share a row, J vectors of V logits each, so that a wave works on 64 / L
// rows at a time, the next ones' logits on their way; its lanes keep the sums of
// their columns' probabilities in registers.  A row's last vector ends with it:
// where V does not divide E it overlaps the one before, and what it has as well
// is not its own: computed alike, stored twice, counted once.
//
// A sum in 32 bits is over at most 16 rows of a lane, the next ones go to another
// and these are added in 64: equal probabilities all round to one side, and one
// sum's error would grow with the tokens.
//
// 32768 tokens of 256 fp32 logits, per call in a graph: 10.3 us for the sums (3.3
// TB/s, where a copy reaches 4.9: a block counts its pairs before its first row's
// softmax, and then has eight rounds alone to hide the loads in), 6.1 for the join
// (a launch, and chains of sixteen loads by a block per 64 experts), 12.0 for the
// gradient (5.6 TB/s, bound by HBM); 61 tokens of 60 in one launch of 4.2,
// gradient 3.0.
#include "elem.h"
#include "lanes.h"

namespace {

using qmoe_lanes::over;

constexpr int kMaxE = 1024;
constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kTerms = 16;    // rows that a lane adds in 32 bits
constexpr int kFinal = 1024;  // threads of the block that finishes

struct Tokens {
  const void* logits;
  const void* ids;      // int32 or int64 [T, k]
  const uint8_t* mask;  // null: every token counts
  int ids64;
  int64_t T;
  int E, k;
};

// Vectors of V elements at any element's address.
template <class T, int V>
struct __attribute__((packed)) Loose {
  typename Vec<T, V>::V v __attribute__((aligned(2)));
};

// A lane's columns: the j-th vector of V at column first(j), of which those from own(j) on are its own.
template <int DT, int V, int L, int J>
struct Row {
  typedef typename Elem<DT>::T T;
  typedef Loose<T, V> Load;
  static constexpr int P = V * J, kRows = 64 / L;  // rows of a wave
  Load raw[J];
  float p[P];
  bool live;

  static __device__ __forceinline__ int own(int j, int lane) { return (lane + j * L) * V; }
  static __device__ __forceinline__ int first(int j, int lane, int E) { return min(own(j, lane), E - V); }
  static __device__ __forceinline__ bool mine(int i, int lane, int E) {
    const int j = i / V;
    return first(j, lane, E) + i % V >= own(j, lane);
  }
  static __device__ __forceinline__ int column(int i, int lane, int E) { return first(i / V, lane, E) + i % V; }

  __device__ __forceinline__ void load(const Tokens& a, int64_t t, int lane) {  // rows past the end: the last again
    const int64_t r = min(t, a.T - 1);
    const T* x = static_cast<const T*>(a.logits) + r * a.E;
    live = t < a.T && (!a.mask || a.mask[r]);
#pragma unroll
    for (int j = 0; j < J; ++j) raw[j] = *reinterpret_cast<const Load*>(x + first(j, lane, a.E));
  }
  __device__ __forceinline__ void softmax(const Tokens& a, int lane) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      p[i] = Elem<DT>::load(at<T, V>(raw[i / V].v, i % V));
      top = fmaxf(top, p[i]);
    }
    top = over<L>(top, [](float x, float y) { return fmaxf(x, y); });
    if (top == -INFINITY) top = 0.f;  // a row of -inf: probabilities of zero
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      p[i] = __expf(p[i] - top);
      sum += mine(i, lane, a.E) ? p[i] : 0.f;
    }
    sum = over<L>(sum, [](float x, float y) { return x + y; });
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < P; ++i) p[i] *= inv;
  }
};

// Counts of this block's share of the pairs, and of its tokens.
__device__ __forceinline__ void count(const Tokens& a, int* counts, int* tokens) {
  const int64_t per = (a.T + gridDim.x - 1) / gridDim.x;  // tokens
  const int64_t t0 = min(per * blockIdx.x, a.T), t1 = min(t0 + per, a.T);
  constexpr int kAhead = 4;
  for (int64_t p = t0 * a.k + threadIdx.x; p < t1 * a.k; p += kAhead * kThreads) {
    int id[kAhead];
    bool live[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t q = min(p + i * kThreads, t1 * a.k - 1);
      const int64_t v = a.ids64 ? static_cast<const int64_t*>(a.ids)[q] : static_cast<const int32_t*>(a.ids)[q];
      id[i] = (int)min(max(v, (int64_t)0), (int64_t)a.E - 1);
      live[i] = p + i * kThreads < t1 * a.k && (!a.mask || a.mask[q / a.k]);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (live[i]) atomicAdd(counts + id[i], 1);
  }
  int n = 0;
  if (a.mask) {
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kThreads) n += a.mask[t] != 0;
  } else if (threadIdx.x == 0) {
    n = (int)(t1 - t0);
  }
  if (n) atomicAdd(tokens, n);
}

struct Result {
  int32_t* counts;
  float* loss;
  int32_t* n;
};
__device__ __forceinline__ void finish(const Result& r, double sum, int n, int E, int k) {
  *r.loss = n ? (float)(sum * E / ((double)n * n * k)) : 0.f;
  *r.n = n;
}

// Rounds of gridDim.x * kWaves * 64 / L rows.  A lone block writes the result itself.
template <int DT, int V, int L, int J>
__global__ __launch_bounds__(kThreads) void balance_sums_kernel(Tokens a, float* __restrict__ psum,
                                                                int32_t* __restrict__ csum, int32_t* __restrict__ nsum,
                                                                int* __restrict__ ticket, Result result) {
  typedef Row<DT, V, L, J> R;
  __shared__ int counts[kMaxE];
  __shared__ float part[kWaves][L * R::P];
  __shared__ double sums[kWaves];
  __shared__ int tokens;
  const int lane = threadIdx.x % L, sub = threadIdx.x % 64 / L, wave = threadIdx.x / 64;
  const int64_t step = (int64_t)gridDim.x * kWaves * R::kRows;
  int64_t t = ((int64_t)blockIdx.x * kWaves + wave) * R::kRows + sub;
  R now, then;
  if (t - sub < a.T) now.load(a, t, lane);
  for (int c = threadIdx.x; c < a.E; c += kThreads) counts[c] = 0;
  if (threadIdx.x == 0) tokens = 0;
  __syncthreads();
  count(a, counts, &tokens);
  float acc[R::P];
  double wide[R::P];
#pragma unroll
  for (int i = 0; i < R::P; ++i) acc[i] = 0.f, wide[i] = 0.0;
  const auto widen = [&] {
#pragma unroll
    for (int i = 0; i < R::P; ++i) wide[i] += acc[i], acc[i] = 0.f;
  };
  bool more = false;
  for (int terms = 0; t - sub < a.T; t += step) {
    if (terms++ == kTerms) widen(), more = true, terms = 1;
    then.load(a, t + step, lane);
    now.softmax(a, lane);
#pragma unroll
    for (int i = 0; i < R::P; ++i) acc[i] += now.live ? now.p[i] : 0.f;
    now = then;
  }
  if (more) {
    widen();
#pragma unroll
    for (int i = 0; i < R::P; ++i) acc[i] = (float)wide[i];
  }
  // the rows that a wave works on at a time, then the waves
#pragma unroll
  for (int i = 0; i < R::P; ++i) {
#pragma unroll
    for (int m = L; m < 64; m *= 2) acc[i] += __shfl_xor(acc[i], m, 64);
    if (sub == 0 && R::mine(i, lane, a.E)) part[wave][R::column(i, lane, a.E)] = acc[i];
  }
  __syncthreads();
  static_assert(kThreads >= kMaxE, "a thread per column");
  const int c = threadIdx.x;
  float v = 0.f;
  if (c < a.E) {
    v = part[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w][c];
  }
  if (gridDim.x > 1) {
    if (c < a.E) {
      psum[(int64_t)blockIdx.x * a.E + c] = v;
      csum[(int64_t)blockIdx.x * a.E + c] = counts[c];
    }
    if (c == 0) nsum[blockIdx.x] = tokens;
    if (blockIdx.x == 0 && c == 0) *ticket = 0;
    return;
  }
  double s = 0.0;
  if (c < a.E) {
    result.counts[c] = counts[c];
    s = (double)v * counts[c];
  }
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) s += __shfl_xor(s, m, 64);
  if (c % 64 == 0) sums[wave] = s;
  __syncthreads();
  if (c) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s += sums[w];
  finish(result, s, tokens, a.E, a.k);
}

// Block b: the blocks' sums of columns 64 b .., sixteen threads to a column, and
// their part of the loss.  The block that is done last (tickets count them) adds
// the parts, in the blocks' order.  One block that reads all sums takes four
// times as long: 256 x 256 of them are half a megabyte.
__global__ __launch_bounds__(kFinal) void balance_loss_kernel(int E, int k, int blocks, const float* __restrict__ psum,
                                                              const int32_t* __restrict__ csum,
                                                              const int32_t* __restrict__ nsum,
                                                              double* parts, int* ticket, Result result) {
  constexpr int kShares = kFinal / 64;
  __shared__ double p[kShares][64];
  __shared__ int c[kShares][64], n;
  const int lane = threadIdx.x % 64, share = threadIdx.x / 64, e = blockIdx.x * 64 + lane;
  if (threadIdx.x == 0) n = 0;
  __syncthreads();
  int live = 0;
  for (int b = threadIdx.x; b < blocks; b += kFinal) live += nsum[b];
  double ps = 0.0;
  int cs = 0;
  if (e < E) {
#pragma unroll 16
    for (int b = share; b < blocks; b += kShares) {
      ps += psum[(int64_t)b * E + e];
      cs += csum[(int64_t)b * E + e];
    }
  }
  if (live) atomicAdd(&n, live);
  p[share][lane] = ps, c[share][lane] = cs;
  __syncthreads();
  if (share) return;
#pragma unroll
  for (int i = 1; i < kShares; ++i) ps += p[i][lane], cs += c[i][lane];
  if (e < E) result.counts[e] = cs;
  double v = e < E ? ps * cs : 0.0;
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) v += __shfl_xor(v, m, 64);
  if (lane) return;
  __hip_atomic_store(parts + blockIdx.x, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // the part is an atomic of the device's scope: once its store is done, every block sees it (a fence would write
  // back and invalidate the caches for the sums' sake, 2 us)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int done = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (done + 1 < (int)gridDim.x) return;
  double sum = 0.0;
  for (int i = 0; i < (int)gridDim.x; ++i) sum += __hip_atomic_load(parts + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  finish(result, sum, n, E, k);
}

template <int DT, int V, int L, int J>
__global__ __launch_bounds__(kThreads) void balance_grad_kernel(Tokens a, const int32_t* __restrict__ counts,
                                                                const int32_t* __restrict__ n_, const float* __restrict__ g,
                                                                void* __restrict__ out_) {
  typedef Row<DT, V, L, J> R;
  const int lane = threadIdx.x % L, sub = threadIdx.x % 64 / L, wave = threadIdx.x / 64;
  const int64_t step = (int64_t)gridDim.x * kWaves * R::kRows;
  int64_t t = ((int64_t)blockIdx.x * kWaves + wave) * R::kRows + sub;
  R now, then;
  if (t - sub < a.T) now.load(a, t, lane);
  const float n = (float)n_[0], fk = n * (float)a.k;
  float f[R::P];
#pragma unroll
  for (int i = 0; i < R::P; ++i) f[i] = (float)counts[R::column(i, lane, a.E)] / fk;
  const float scale = *g * (float)a.E / n;
  for (; t - sub < a.T; t += step) {
    then.load(a, t + step, lane);
    now.softmax(a, lane);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < R::P; ++i) dot += R::mine(i, lane, a.E) ? f[i] * now.p[i] : 0.f;
    dot = over<L>(dot, [](float x, float y) { return x + y; });
    if (t < a.T) {
      typename R::T* out = static_cast<typename R::T*>(out_) + t * a.E;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (R::own(j, lane) >= a.E) break;
        typename R::Load o;
#pragma unroll
        for (int i = 0; i < V; ++i)
          set<typename R::T, V>(o.v, i, Elem<DT>::store(now.live ? scale * (now.p[j * V + i] * (f[j * V + i] - dot)) : 0.f));
        *reinterpret_cast<typename R::Load*>(out + R::first(j, lane, a.E)) = o;
      }
    }
    now = then;
  }
}

// Lanes per row of E logits.
int lanes_of(int64_t E) {
  int L = 4;
  while (L < 64 && 4 * L < E) L *= 2;
  return L;
}
// Blocks of the sums: one for up to four rounds, which needs no second launch,
// else of two rounds each at least, and one per CU at most.
int64_t blocks_of(int64_t T, int64_t E) {
  const int64_t rows = kWaves * (64 / lanes_of(E)), b = (T + 2 * rows - 1) / (2 * rows);
  return T <= 4 * rows ? 1 : b > 256 ? 256 : b;
}

struct Sums {
  Tokens a;
  float* psum;
  int32_t *csum, *nsum;
  int* ticket;
  Result result;
  hipStream_t st;
  template <int DT, int V, int L, int J>
  void run() const {
    balance_sums_kernel<DT, V, L, J><<<dim3((unsigned)blocks_of(a.T, a.E)), dim3(kThreads), 0, st>>>(a, psum, csum, nsum, ticket, result);
  }
};
struct Grad {
  Tokens a;
  const int32_t *counts, *n;
  const float* g;
  void* out;
  hipStream_t st;
  template <int DT, int V, int L, int J>
  void run() const {
    const int64_t rows = kWaves * (64 / L), blocks = (a.T + rows - 1) / rows;
    const dim3 grid((unsigned)(blocks > 512 ? 512 : blocks));
    balance_grad_kernel<DT, V, L, J><<<grid, dim3(kThreads), 0, st>>>(a, counts, n, g, out);
  }
};
// The form of a row of E logits.
template <int DT, class Run>
void with_form(const Run& run, int E) {
  if (E < 4) return run.template run<DT, 1, 4, 1>();
  switch (lanes_of(E)) {
    case 4: return run.template run<DT, 4, 4, 1>();
    case 8: return run.template run<DT, 4, 8, 1>();
    case 16: return run.template run<DT, 4, 16, 1>();
    case 32: return run.template run<DT, 4, 32, 1>();
    default: break;
  }
  if (E <= 256) run.template run<DT, 4, 64, 1>();
  else if (E <= 512) run.template run<DT, 4, 64, 2>();
  else run.template run<DT, 4, 64, 4>();
}
template <class Run>
void with_type(const Run& run, int dtype, int E) {
  if (dtype == QMOE_BF16) with_form<QMOE_BF16>(run, E);
  else if (dtype == QMOE_FP16) with_form<QMOE_FP16>(run, E);
  else with_form<QMOE_FP32>(run, E);
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
  // parts of the loss, sums, counts and tokens by block, the ticket
  return sizeof(double) * (kMaxE / 64) + 4 * ((size_t)blocks_of(T, E) * (2 * E + 1) + 1);
}

extern "C" int qmoe_router_balance(const void* logits, int dtype, int64_t T, int64_t E, const void* ids, int ids64,
                                   int64_t k, const uint8_t* mask, float* loss, int32_t* counts, int32_t* n,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const Tokens a{logits, ids, mask, ids64, T, (int)E, (int)k};
  const int rc = check(a, E, k, dtype, true);
  if (rc != QMOE_OK) return rc;
  if (!loss || !counts || !n) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "the workspace must be 8-byte aligned");
  if (!workspace || workspace_bytes < qmoe_router_balance_workspace_size(T, E))
    return qmoe::fail(QMOE_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", workspace_bytes,
                      qmoe_router_balance_workspace_size(T, E));
  const int blocks = (int)blocks_of(T, E);
  double* parts = static_cast<double*>(workspace);
  float* psum = reinterpret_cast<float*>(parts + kMaxE / 64);
  int32_t* csum = reinterpret_cast<int32_t*>(psum + (size_t)blocks * E);
  int32_t* nsum = csum + (size_t)blocks * E;
  hipStream_t st = qmoe::as_stream(stream);
  int* ticket = nsum + blocks;
  const Result result{counts, loss, n};
  with_type(Sums{a, psum, csum, nsum, ticket, result, st}, dtype, a.E);
  if (const int rc2 = qmoe::launch_status("balance_sums_kernel")) return rc2;
  if (blocks == 1) return QMOE_OK;
  balance_loss_kernel<<<dim3((unsigned)((E + 63) / 64)), dim3(kFinal), 0, st>>>(a.E, a.k, blocks, psum, csum, nsum, parts,
                                                                               ticket, result);
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
  with_type(Grad{a, counts, n, dloss, dlogits, qmoe::as_stream(stream)}, dtype, a.E);
  return qmoe::launch_status("balance_grad_kernel");
}
