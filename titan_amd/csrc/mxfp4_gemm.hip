// Products of mxfp4 weights with many rows on the matrix cores: bf16
// activations either way round (x W^T over the packed axis, x W over the
// rows), and activations in mxfp4 too (format in mxfp4.h).  Rows are those of
// a tile table (sorted by expert), or of one expert without a table.
#include "gemm_common.h"
#include "mxfp4.h"

namespace {

using namespace qmoe_mx;
using qmoe_gemm::kTileRows;

enum { kFwd = 0, kT = 1, kQQ = 2 };

struct GemmArgs {
  const uint16_t* x;     // bf16 rows, ldx elements apart
  const uint32_t* xq;    // kQQ: codes [n_x, K/8]
  const uint8_t* xs;     // kQQ: scales [n_x, K/32]
  const int32_t* x_rows;
  int64_t n_rows, n_x, ldx;
  const uint32_t* w;
  const uint8_t* s;
  int num_experts;
  int64_t N, K;
  const int32_t *offsets, *tile_row, *tile_exp, *ntiles;  // all null: one expert, rows in order
  void* out;
  int out_f32;
};

__device__ __forceinline__ qmoe_gemm::TileRows tile_of(const GemmArgs& a, int64_t tile) {
  if (a.offsets) {
    qmoe_gemm::TileRows t{0, 0, 0};
    if (tile >= a.ntiles[0]) return t;
    const qmoe_gemm::Tiles tiles{a.offsets, a.tile_row, a.tile_exp, a.ntiles, a.n_rows, a.num_experts};
    return qmoe_gemm::tile_rows_of(tiles, (int)tile);
  }
  qmoe_gemm::TileRows t;
  t.e = 0;
  t.row0 = tile * kTileRows;
  t.valid = (int)max((int64_t)0, min((int64_t)kTileRows, a.n_rows - t.row0));
  return t;
}

constexpr int kStep = 32, kOut = 64, kPitch = kStep + 8;

template <int MODE>
__global__ __launch_bounds__(256) void mx_gemm_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t xa[kTileRows][kPitch];
  __shared__ __attribute__((aligned(16))) uint16_t wb[kOut][kPitch];
  const qmoe_gemm::TileRows t = tile_of(a, blockIdx.x);
  if (t.valid <= 0) return;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int64_t C = MODE == kT ? a.N : a.K, O = MODE == kT ? a.K : a.N;
  const int64_t o0 = (int64_t)blockIdx.y * kOut;
  const int64_t units = a.K / kBlock;
  f32x4_t acc[2][4] = {};
  for (int64_t c0 = 0; c0 < C; c0 += kStep) {
    __syncthreads();
    for (int i = tid; i < kTileRows * 4; i += 256) {
      const int m = i / 4, u = i % 4;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (m < t.valid && c0 + 8 * u < C) {
        const int64_t r = t.row0 + m;
        const int64_t xr = min(max(a.x_rows ? (int64_t)a.x_rows[r] : r, (int64_t)0), a.n_x - 1);
        if constexpr (MODE == kQQ) {
          uint32_t p[4];
          unpack8(a.xq[xr * 4 * units + c0 / 8 + u], scale_of(a.xs[xr * units + c0 / kBlock]), p);
          v = make_uint4(p[0], p[1], p[2], p[3]);
        } else {
          v = *reinterpret_cast<const uint4*>(a.x + xr * a.ldx + c0 + 8 * u);
        }
      }
      *reinterpret_cast<uint4*>(&xa[m][8 * u]) = v;
    }
    {
      uint32_t p[4] = {0, 0, 0, 0};
      if constexpr (MODE == kT) {
        const int n = tid / 8, j = tid % 8;  // weight row of the step, word of its 64 outputs
        if (c0 + n < C && o0 + 8 * j < O) {
          const int64_t row = (int64_t)t.e * a.N + c0 + n;
          unpack8(a.w[row * 4 * units + o0 / 8 + j], scale_of(a.s[row * units + (o0 + 8 * j) / kBlock]), p);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) wb[8 * j + i][n] = (uint16_t)(p[i / 2] >> (16 * (i & 1)));
      } else {
        const int n = tid / 4, j = tid % 4;
        if (o0 + n < O) {
          const int64_t row = (int64_t)t.e * a.N + o0 + n;
          unpack8(a.w[row * 4 * units + c0 / 8 + j], scale_of(a.s[row * units + c0 / kBlock]), p);
        }
        *reinterpret_cast<uint4*>(&wb[n][8 * j]) = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
    __syncthreads();
    bf16x8_t fa[2], fb[4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      fa[i] = *reinterpret_cast<const bf16x8_t*>(&xa[32 * wave + 16 * i + lane % 16][8 * (lane / 16)]);
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[j] = *reinterpret_cast<const bf16x8_t*>(&wb[16 * j + lane % 16][8 * (lane / 16)]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = 32 * wave + 16 * i + lane % 16;
        const int64_t o = o0 + 16 * j + 4 * (lane / 16) + q;
        if (m >= t.valid || o >= O) continue;
        const int64_t at = (t.row0 + m) * O + o;
        if (a.out_f32) static_cast<float*>(a.out)[at] = acc[i][j][q];
        else static_cast<uint16_t*>(a.out)[at] = (uint16_t)f32_to_bf16(acc[i][j][q]);
      }
}

template <int MODE>
int launch(GemmArgs a, int64_t max_tiles, hipStream_t st) {
  const int64_t O = MODE == kT ? a.K : a.N;
  const int64_t tiles = a.offsets ? max_tiles : (a.n_rows + kTileRows - 1) / kTileRows;
  const int64_t cols = (O + kOut - 1) / kOut;
  if (tiles > 0x7FFFFFFF || cols > 65535) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  mx_gemm_kernel<MODE><<<dim3((unsigned)tiles, (unsigned)cols), dim3(256), 0, st>>>(a);
  return qmoe::launch_status("mx_gemm_kernel");
}

// Argument checks shared by the entry points; QMOE_OK with *run = false: nothing to do.
int check(const GemmArgs& a, int mode, int64_t max_tiles, int out_dtype, bool* run) {
  *run = false;
  if (a.n_rows < 0 || a.n_x < 0 || a.N < 0 || a.K < 0 || a.num_experts < 0 || max_tiles < 0)
    return qmoe::fail(QMOE_ERR_INVALID, "bad sizes");
  if (out_dtype != QMOE_BF16 && out_dtype != QMOE_FP32)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "out_dtype=%d", out_dtype);
  if (a.K % kBlock) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "K=%lld: must be a multiple of 32", (long long)a.K);
  const int64_t C = mode == kT ? a.N : a.K, O = mode == kT ? a.K : a.N;
  if (a.n_rows == 0 || O == 0) return QMOE_OK;
  if (C == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty contraction");
  if (a.n_x == 0 || a.num_experts == 0) return qmoe::fail(QMOE_ERR_INVALID, "no activation rows or no experts");
  if (!a.w || !a.s || !a.out || (mode == kQQ ? !a.xq || !a.xs : !a.x)) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  const bool any = a.offsets || a.tile_row || a.tile_exp || a.ntiles;
  if (any && !(a.offsets && a.tile_row && a.tile_exp && a.ntiles)) return qmoe::fail(QMOE_ERR_INVALID, "half a tile table");
  if (!any && a.num_experts != 1) return qmoe::fail(QMOE_ERR_INVALID, "several experts need a tile table");
  if (!any && !a.x_rows && a.n_x < a.n_rows) return qmoe::fail(QMOE_ERR_INVALID, "fewer activation rows than rows");
  if (any && max_tiles == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty tile table");
  if (a.N > 0x7FFFFFFF || a.K > 0x7FFFFFFF || a.n_rows > 0x7FFFFFFF || a.n_x > 0x7FFFFFFF || max_tiles > 0x7FFFFFFF)
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  if (!qmoe::aligned16(a.w) || !qmoe::aligned16(a.out)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "codes and out must be 16-byte aligned");
  if (mode == kQQ ? !qmoe::aligned16(a.xq) : (!qmoe::aligned16(a.x) || a.ldx % 8 || a.ldx < C))
    return qmoe::fail(QMOE_ERR_UNSUPPORTED, "activation rows must be 16-byte aligned and at least as long as the contraction");
  *run = true;
  return QMOE_OK;
}

}  // namespace

extern "C" int qmoe_mxfp4_gather_qmm(const uint16_t* x, int64_t n_x, int64_t ldx, const int32_t* x_rows, int64_t n_rows,
                                     const uint32_t* w, const uint8_t* scales, int32_t num_experts, int64_t N,
                                     int64_t K, int transpose, const int32_t* offsets, const int32_t* tile_row,
                                     const int32_t* tile_exp, const int32_t* ntiles, int64_t max_tiles, int out_dtype,
                                     void* out, void* stream) {
  GemmArgs a{x, nullptr, nullptr, x_rows, n_rows, n_x, ldx, w, scales, num_experts, N, K,
             offsets, tile_row, tile_exp, ntiles, out, out_dtype == QMOE_FP32};
  bool run;
  const int rc = check(a, transpose ? kFwd : kT, max_tiles, out_dtype, &run);
  if (rc != QMOE_OK || !run) return rc;
  hipStream_t st = qmoe::as_stream(stream);
  return transpose ? launch<kFwd>(a, max_tiles, st) : launch<kT>(a, max_tiles, st);
}

extern "C" int qmoe_mxfp4_gather_qqmm(const uint32_t* xq, const uint8_t* xs, int64_t n_x, const int32_t* x_rows,
                                      int64_t n_rows, const uint32_t* w, const uint8_t* scales, int32_t num_experts,
                                      int64_t N, int64_t K, const int32_t* offsets, const int32_t* tile_row,
                                      const int32_t* tile_exp, const int32_t* ntiles, int64_t max_tiles, void* out,
                                      void* stream) {
  GemmArgs a{nullptr, xq, xs, x_rows, n_rows, n_x, 0, w, scales, num_experts, N, K,
             offsets, tile_row, tile_exp, ntiles, out, 0};
  bool run;
  const int rc = check(a, kQQ, max_tiles, QMOE_BF16, &run);
  if (rc != QMOE_OK || !run) return rc;
  return launch<kQQ>(a, max_tiles, qmoe::as_stream(stream));
}
