// Products of one matrix of 8-bit integers with a few rows (int8_product.h),
// every weight read once for 16 or 32 of them: from HBM the first time, by more
// rows from the caches.
//
// A block owns 16 outputs of 16 * MT rows, and its eight waves take batches of
// BK of the contraction in turn; their partial sums meet in LDS at the end and
// are added.  A wave copies its batch, whole lines of each row, into a buffer of
// its own, so nothing waits on a barrier, and with K = 2048 all of a call's
// bytes are requested in one or two rounds.  Lane (n = lane % 16, q = lane / 16)
// holds sixteen codes of row n, 64 of a row at a time go through
// v_mfma_i32_16x16x64_i8.
//
// Bound by a launch, one or two rounds of dependent copies and the join: 4096 x
// 2048 weights, per call in a graph, 5 rows 5.0 us, 32 rows 5.8, 64 rows 6.9
// (8.4 MB: 1.7 at a copy's rate).
#include "gemm_common.h"
#include "int8_few.h"

namespace {

using namespace qmoe_i8;
using qmoe_gemm::dma16;

constexpr int kWaves = 8;
__device__ __attribute__((aligned(16))) uint32_t zero_unit[4];  // what copies past the contraction's end read

// Swizzle of a row's 16-byte units in LDS, UNITS of them: one unit of sixteen rows at a time is read from all banks.
template <int UNITS>
__device__ __forceinline__ int swz(int row) {
  return UNITS <= 8 ? (row >> 1) & (UNITS - 1) : row & 15;
}

// Copies 16 rows of UNITS 16-byte units each, from unit u0 of every row, into
// LDS, swizzled; units from `units` on are zeros.
template <int UNITS>
__device__ __forceinline__ void copy_rows(const char* (&row)[UNITS / 4], int u0, int units, uint32_t dst, int lane) {
  constexpr int kPer = 64 / UNITS;  // rows per copy
#pragma unroll
  for (int d = 0; d < UNITS / 4; ++d) {
    const int u = (lane % UNITS) ^ swz<UNITS>(d * kPer + lane / UNITS);
    const char* p = row[d] + (size_t)(u0 + u) * 16;
    dma16(u0 + u < units ? p : reinterpret_cast<const char*>(zero_unit), dst + d * 1024);
  }
}

template <int MT, int BK>
__global__ __launch_bounds__(64 * kWaves) void int8_few_kernel(Product a) {
  constexpr int kUnits = BK / 16, kPer = 64 / kUnits;
  constexpr int kTile = 16 * BK, kBuf = (1 + MT) * kTile, kSums = kWaves * MT * 256 * 4;
  constexpr int kLds = kWaves * kBuf > kSums ? kWaves * kBuf : kSums;
  static_assert(kLds <= 160 * 1024, "LDS per CU");
  __shared__ __attribute__((aligned(16))) char smem[kLds];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int n16 = lane % 16, q = lane / 16;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
  const int units = (int)(a.K / 16);
  const auto x_row = [&](int64_t m) {  // rows past the end: the last again, not stored
    const int64_t r = min(m0 + m, a.n_rows - 1);
    return min(max(a.x_rows ? (int64_t)a.x_rows[r] : r, (int64_t)0), a.n_x - 1);
  };
  const char *w[kUnits / 4], *x[MT][kUnits / 4];
#pragma unroll
  for (int d = 0; d < kUnits / 4; ++d) {
    const int r = d * kPer + lane / kUnits;
    w[d] = reinterpret_cast<const char*>(a.w) + min(n0 + r, a.N - 1) * a.K;
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t][d] = reinterpret_cast<const char*>(a.x) + x_row(16 * t + r) * a.K;
  }
  char* buf = smem + wave * kBuf;
  const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)buf);
  i32x4_t acc[MT] = {};
  const int batches = (int)((a.K + BK - 1) / BK);
  for (int b = wave; b < batches; b += kWaves) {
    copy_rows<kUnits>(w, b * kUnits, units, lds, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t) copy_rows<kUnits>(x[t], b * kUnits, units, lds + (1 + t) * kTile, lane);
    qmoe_gemm::wait_vmem<0>();
#pragma unroll
    for (int c = 0; c < BK / 64; ++c) {
      const int at = n16 * BK + ((4 * c + q) ^ swz<kUnits>(n16)) * 16;
      const i32x4_t wv = *reinterpret_cast<const i32x4_t*>(buf + at);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const i32x4_t xv = *reinterpret_cast<const i32x4_t*>(buf + (1 + t) * kTile + at);
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv, acc[t], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer is read before the next batch is copied into it
  }
  __syncthreads();
  // partial sums [wave][row][16 outputs]: a lane holds outputs 4q .. 4q + 3 of row n16 of each tile
  int* sums = reinterpret_cast<int*>(smem);
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<i32x4_t*>(sums + ((wave * MT + t) * 16 + n16) * 16 + 4 * q) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += 64 * kWaves) {
    const int64_t m = m0 + i / 16, n = n0 + i % 16;
    int v = 0;
#pragma unroll
    for (int j = 0; j < kWaves; ++j) v += sums[j * MT * 256 + i];
    if (m < a.n_rows && n < a.N) put(a, m * a.N + n, scaled(v, a.sx[x_row(i / 16)], a.sw[n]));
  }
}

template <int MT, int BK>
int launch(const Product& a, hipStream_t st) {
  // blocks of the same weights on the same XCD, as in int8_qmv.hip (64 rows by 1000 of 4096: 6.4 -> 5.2 us); what is
  // past the end works on the last weight row
  const int64_t rows = (a.n_rows + 16 * MT - 1) / (16 * MT), cols = (a.N + 15) / 16;
  const dim3 grid((unsigned)(rows > 1 ? (cols + 7) / 8 * 8 : cols), (unsigned)rows);
  if (qmoe::too_many((int64_t)grid.x * grid.y, 64 * kWaves))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "N=%lld: too large", (long long)a.N);
  int8_few_kernel<MT, BK><<<grid, dim3(64 * kWaves), 0, st>>>(a);
  return qmoe::launch_status("int8_few_kernel");
}

}  // namespace

// 16 rows a block where that makes no more blocks than 32 would, or no more than
// the chip has CUs; else 32. (16 / 32, us per call in a graph: 4096 x 2048 weights,
// 16 rows 5.2 / 5.4, 64 rows 8.0 / 6.9; 1024 x 4096, 64 rows 5.0 / 5.7, 96 rows 6.0 /
// 5.7. 32 rows by 32 outputs: 6.5, 6.9 and 6.8 there.)
int qmoe_i8::few_product(const Product& a, hipStream_t st) {
  const int64_t blocks = (a.n_rows + 15) / 16 * ((a.N + 15) / 16);
  return a.n_rows <= 16 || blocks <= 256 ? launch<1, 256>(a, st) : launch<2, 128>(a, st);
}
