// Products of one matrix of mxfp4 weights with a few rows (5 to 64), bf16 or
// mxfp4: out[m, n] = sum_k x[m, k] W[n, k], every weight read once (format in
// mxfp4.h).
//
// A block owns 16 outputs of 16 * MT rows, and its eight waves take batches of
// BK of the contraction in turn; their partial sums meet in LDS at the end and
// are added in wave order.  A wave copies its batch's codes and activations,
// whole lines of each row, into a buffer of its own (read straight into the
// matrix instructions' layout, 16 rows under 16 neighbouring lanes, a load
// costs its lanes a cycle each), so nothing waits on a barrier, and with K =
// 2048 all of a call's bytes are requested in one or two rounds.  Lane (n = lane % 16, q =
// lane / 16) holds block q of four of row n: v_mfma_f32_16x16x32_bf16 takes a
// word of it at a time, converted, against the same columns of x;
// v_mfma_scale_f32_16x16x128_f8f6f4 (QQ) the block as it is against x's codes.
//
// Bound by the two or three dependent round trips to HBM of a launch: 4096 x
// 2048 weights (4.5 MB) take 4.8 us per call in a graph at 5 rows, 6.4 at 32,
// 8.7 at 64.
#include "gemm_common.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"

namespace {

using namespace qmoe_mx;
using qmoe_gemm::dma16;

constexpr int kWaves = 8;
__device__ __attribute__((aligned(16))) uint32_t zero_unit[4];  // what copies past the contraction's end read

// Swizzles of a row's 16-byte units in LDS: one unit of sixteen rows at a time
// is read from all banks, for rows of 8 or fewer units and of 16 or more.
__device__ __forceinline__ int swz_short(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz_long(int row) { return row & 15; }

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;

template <bool QQ, int MT, int BK>
struct Cfg {
  static constexpr int kChunks = BK / 128;
  static constexpr int kW = 16 * BK / 2;                           // codes of 16 rows
  static constexpr int kX = QQ ? MT * kW : MT * 16 * BK * 2;       // activations of 16 * MT rows
  static constexpr int kBuf = kW + kX;
  static constexpr int kSums = kWaves * MT * 16 * 16 * 4;
  static constexpr int kLds = kWaves * kBuf > kSums ? kWaves * kBuf : kSums;
  static_assert(kLds <= 160 * 1024, "LDS per CU");
};

// Copies 16 rows of UNITS 16-byte units each, from unit u0 of every row, into
// LDS, swizzled; units from `units` on are zeros.
template <int UNITS>
__device__ __forceinline__ void copy_rows(const char* (&row)[UNITS / 4], int u0, int units, uint32_t dst, int lane) {
  constexpr int kPer = 64 / UNITS;  // rows per copy
#pragma unroll
  for (int d = 0; d < UNITS / 4; ++d) {
    const int r = d * kPer + lane / UNITS;
    const int u = (lane % UNITS) ^ (UNITS <= 8 ? swz_short(r) & (UNITS - 1) : swz_long(r));
    const char* p = row[d] + (size_t)(u0 + u) * 16;
    dma16(u0 + u < units ? p : reinterpret_cast<const char*>(zero_unit), dst + d * 1024);
  }
}
// The base of each copy's row for this lane.
template <int UNITS, class F>
__device__ __forceinline__ void row_bases(const char* (&row)[UNITS / 4], int lane, F base) {
  constexpr int kPer = 64 / UNITS;
#pragma unroll
  for (int d = 0; d < UNITS / 4; ++d) row[d] = base(d * kPer + lane / UNITS);
}

template <bool QQ, int MT, int BK>
__global__ __launch_bounds__(64 * kWaves) void mx_rows_kernel(RowsArgs a) {
  typedef Cfg<QQ, MT, BK> C;
  constexpr int kWUnits = BK / 32, kXUnits = QQ ? BK / 32 : BK / 8;
  __shared__ __attribute__((aligned(16))) char smem[C::kLds];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  const int n16 = lane % 16, q = lane / 16;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
  const int units = (int)(a.K / kBlock), xunits = QQ ? units : units * 4;
  const auto x_row = [&](int64_t m) {  // rows past the end: the last again, not stored
    const int64_t r = min(m0 + m, a.M - 1);
    return min(max(a.x_rows ? (int64_t)a.x_rows[r] : r, (int64_t)0), a.n_x - 1);
  };
  const char* w[kWUnits / 4];
  row_bases<kWUnits>(w, lane, [&](int r) {
    return reinterpret_cast<const char*>(a.w) + min(n0 + r, a.N - 1) * units * 16;
  });
  const char* x[MT][kXUnits / 4];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    row_bases<kXUnits>(x[t], lane, [&](int r) {
      const int64_t row = x_row(16 * t + r);
      return QQ ? reinterpret_cast<const char*>(a.xq) + row * units * 16 : reinterpret_cast<const char*>(a.x) + row * a.ldx * 2;
    });
  const uint8_t* ws = a.s + min(n0 + n16, a.N - 1) * units;
  const uint8_t* xs[MT];
  if constexpr (QQ) {
#pragma unroll
    for (int t = 0; t < MT; ++t) xs[t] = a.xs + x_row(16 * t + n16) * units;
  }
  char* buf = smem + wave * C::kBuf;
  const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)buf);
  f32x4_t acc[MT] = {};
  const int batches = (int)((a.K + BK - 1) / BK);
  for (int b = wave; b < batches; b += kWaves) {
    const int u0 = b * (BK / kBlock);
    // a block past the end has scale byte 0: its codes are zeros
    uint32_t sb[C::kChunks], xb[MT][C::kChunks];
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) {
      const int u = u0 + 4 * c + q;
      sb[c] = u < units ? ws[u] : 0u;
      if constexpr (QQ) {
#pragma unroll
        for (int t = 0; t < MT; ++t) xb[t][c] = u < units ? xs[t][u] : 0u;
      }
    }
    copy_rows<kWUnits>(w, u0, units, lds, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t)
      copy_rows<kXUnits>(x[t], QQ ? u0 : 4 * u0, xunits, lds + C::kW + t * (C::kX / MT), lane);
    qmoe_gemm::wait_vmem<0>();
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c) {
      const int wu = (4 * c + q) ^ (swz_short(n16) & (kWUnits - 1));
      const i32x4_t codes = *reinterpret_cast<const i32x4_t*>(buf + n16 * kWUnits * 16 + wu * 16);
      if constexpr (QQ) {
        const i32x8_t wide = {codes[0], codes[1], codes[2], codes[3], 0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const i32x4_t v = *reinterpret_cast<const i32x4_t*>(buf + C::kW + t * C::kW + n16 * kWUnits * 16 + wu * 16);
          const i32x8_t xw = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, xw, acc[t], 4, 4, 0, (int)sb[c], 0, (int)xb[t][c]);
        }
      } else {
        const float sc = scale_of(sb[c]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t p[4];
          unpack8((uint32_t)codes[kk], sc, p);
          const i32x4_t wf = {(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
          const int xu = (16 * c + 4 * q + kk) ^ swz_long(n16);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const i32x4_t v = *reinterpret_cast<const i32x4_t*>(buf + C::kW + t * (C::kX / MT) + n16 * kXUnits * 16 + xu * 16);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, wf),
                                                             __builtin_bit_cast(bf16x8_t, v), acc[t], 0, 0, 0);
          }
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer is read before the next batch is copied into it
  }
  __syncthreads();
  // partial sums [wave][row][16 outputs]: a lane holds outputs 4q .. 4q + 3 of row n16 of each tile
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < MT; ++t)
    *reinterpret_cast<f32x4_t*>(sums + ((wave * MT + t) * 16 + n16) * 16 + 4 * q) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += 64 * kWaves) {
    const int64_t m = m0 + i / 16, n = n0 + i % 16;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < kWaves; ++j) v += sums[j * MT * 256 + i];
    if (m >= a.M || n >= a.N) continue;
    if (a.out_f32) static_cast<float*>(a.out)[m * a.N + n] = v;
    else static_cast<uint16_t*>(a.out)[m * a.N + n] = (uint16_t)f32_to_bf16(v);
  }
}

template <bool QQ, int MT, int BK>
int launch(const RowsArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  if (qmoe::too_many((int64_t)grid.x * grid.y, 64 * kWaves))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "N=%lld: too large", (long long)a.N);
  mx_rows_kernel<QQ, MT, BK><<<grid, dim3(64 * kWaves), 0, st>>>(a);
  return qmoe::launch_status("mx_rows_kernel");
}

}  // namespace

int qmoe_mx::rows_product(const RowsArgs& a, bool qq, hipStream_t st) {
  // Row tiles of 16 as many as there are rows for.  Batches of 256 where two blocks still fit a CU: with one, blocks
  // past the 256th wait for a round of their own (us per call in a graph, 23 rows, batches of 256 / 128: 4099 x 2080 10.2 / 6.8 us, 8192 x
  // 2048 10.7 / 7.6, 4096 x 2048 6.2 / 5.6; in smaller forms either is within 8% of the other).
  const int mt = (int)((a.M + 15) / 16);
  if (qq) {
    if (mt <= 1) return launch<true, 1, 256>(a, st);
    return mt == 2 ? launch<true, 2, 256>(a, st) : launch<true, 4, 256>(a, st);
  }
  if (mt <= 1) return launch<false, 1, 256>(a, st);
  if (mt == 2) return launch<false, 2, 128>(a, st);
  return mt == 3 ? launch<false, 3, 128>(a, st) : launch<false, 4, 128>(a, st);
}
