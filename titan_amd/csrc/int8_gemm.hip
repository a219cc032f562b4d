// Products of 8-bit integers with many rows on the matrix cores
// (int8_product.h).  Rows are those of a tile table (sorted by expert), or of
// one expert without a table.
#include "gemm_common.h"
#include "int8_product.h"

namespace {

using namespace qmoe_i8;
using qmoe_gemm::kTileRows;

// One wave per 32 rows of a tile and 32 outputs, operands straight from memory.
__global__ __launch_bounds__(64) void int8_tile_kernel(Product a) {
  const int lane = threadIdx.x, l32 = lane % 32, h = lane / 32;
  const int64_t tile = blockIdx.y / 4, sub = blockIdx.y % 4, n0 = (int64_t)blockIdx.x * 32;
  int64_t row0 = tile * kTileRows, valid = a.n_rows - row0;
  int64_t e = 0;
  if (a.offsets) {
    if (tile >= a.ntiles[0]) return;
    const qmoe_gemm::Tiles t{a.offsets, a.tile_row, a.tile_exp, a.ntiles, a.n_rows, a.num_experts};
    const qmoe_gemm::TileRows tr = qmoe_gemm::tile_rows_of(t, (int)tile);
    row0 = tr.row0, valid = tr.valid, e = tr.e;
  }
  row0 += 32 * sub, valid -= 32 * sub;
  if (valid <= 0) return;
  const int64_t xr = x_row_of(a, row0 + min((int64_t)l32, valid - 1));
  const int64_t n = e * a.N + min(n0 + l32, a.N - 1);
  i32x16_t acc = {};
  for (int64_t k = 16 * h; k < a.K + 16 * h; k += 32) {
    const i32x4_t zero = {};
    const i32x4_t xv = k < a.K ? *reinterpret_cast<const i32x4_t*>(a.x + xr * a.K + k) : zero;
    const i32x4_t wv = k < a.K ? *reinterpret_cast<const i32x4_t*>(a.w + n * a.K + k) : zero;
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wv, xv, acc, 0, 0, 0);
  }
  if (l32 >= valid) return;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t o = n0 + 8 * (v / 4) + 4 * h + v % 4;
    if (o < a.N) put(a, (row0 + l32) * a.N + o, scaled(acc[v], a.sx[xr], a.sw[e * a.N + o]));
  }
}

}  // namespace

extern "C" int qmoe_int8_gather_qqmm(const int8_t* x, const float* sx, int64_t n_x, const int32_t* x_rows, int64_t n_rows,
                                     const int8_t* w, const float* sw, int32_t num_experts, int64_t N, int64_t K,
                                     const int32_t* offsets, const int32_t* tile_row, const int32_t* tile_exp,
                                     const int32_t* ntiles, int64_t max_tiles, int out_dtype, void* out, void* stream) {
  Product a{x, sx, x_rows, n_rows, n_x, 1, nullptr, w, sw, num_experts, N, K, offsets, tile_row, tile_exp, ntiles, out, out_dtype};
  bool run;
  const int rc = check(a, &run);
  if (rc != QMOE_OK || !run) return rc;
  const bool any = offsets || tile_row || tile_exp || ntiles;
  if (any && !(offsets && tile_row && tile_exp && ntiles)) return qmoe::fail(QMOE_ERR_INVALID, "half a tile table");
  if (!any && num_experts != 1) return qmoe::fail(QMOE_ERR_INVALID, "several experts need a tile table");
  if (!any && !x_rows && n_x < n_rows) return qmoe::fail(QMOE_ERR_INVALID, "fewer activation rows than rows");
  if (any && max_tiles <= 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty tile table");
  if (max_tiles > 0x7FFFFFFF) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  const int64_t tiles = any ? max_tiles : (n_rows + kTileRows - 1) / kTileRows;
  const dim3 grid((unsigned)((N + 31) / 32), (unsigned)(4 * tiles));
  if (4 * tiles > 65535 || qmoe::too_many((int64_t)grid.x * grid.y, 64)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "too many rows");
  int8_tile_kernel<<<grid, dim3(64), 0, qmoe::as_stream(stream)>>>(a);
  return qmoe::launch_status("int8_tile_kernel");
}
