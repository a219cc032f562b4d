// Products of 8-bit integers with many rows on the matrix cores
// (int8_product.h).  Rows are those of a tile table (sorted by expert), or of
// one expert without a table.
//
// A unit is a block of up to kRows rows of one expert times kCols outputs.  Its
// WM x WN waves hold MSUB x NSUB subtiles of v_mfma_i32_32x32x32_i8 each.  Both
// operands reach LDS by asynchronous copies into a ring of NS stages of KB
// bytes of the contraction, and are read from there as fragments, those of a
// step during the step before.  The barrier that hands over a stage stands
// before a group's last step, whose operands are in registers by then; the
// copies into the stage that it frees are spread between the matrix
// instructions that follow, since a run of them would hold up the wave that
// issues them.  Blocks are persistent; units of a table go heavy-first
// (gemm_common.h), those of one matrix in bands of columns, so that the blocks
// of an XCD share rows and columns in its L2.
#include <algorithm>

#include "gemm_common.h"
#include "int8_product.h"

namespace {

using namespace qmoe_i8;
using qmoe_gemm::kTileRows;

constexpr int kLdsCU = 160 * 1024;
__device__ __attribute__((aligned(16))) uint32_t zero_unit[4];  // what copies past the contraction's end read

// The thread's index through an empty asm, so that what is computed from it is
// computed here and not kept in registers across the unit loop.
__device__ __forceinline__ int fresh_tid() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

struct Unit {
  int e, valid;
  int64_t row0, o0;  // first row; first output
};

// The activation row of a unit's row; past the end: the last again, not stored.
__device__ __forceinline__ int64_t row_of(const Product& a, const Unit& u, int row) {
  const int64_t r = u.row0 + min(row, u.valid - 1);
  return min(max(a.x_rows ? (int64_t)a.x_rows[r] : r, (int64_t)0), a.n_x - 1);
}

// Swizzle of a row's 16-byte units in LDS, KB / 16 of them: one unit of sixteen
// consecutive rows is read without bank conflicts.
template <int KB>
__device__ __forceinline__ int swz(int row) {
  if constexpr (KB == 128) return (row & 7) ^ ((row >> 3) & 1);
  else return (row >> 2) & 3;
}

// Sixteen bytes stored at any element's address.
struct __attribute__((packed)) Loose16 {
  i32x4_t v __attribute__((aligned(2)));
};

template <int WM_, int WN_, int MSUB_, int NSUB_, int KB_, int NS_>
struct Form {
  static constexpr int WM = WM_, WN = WN_, MSUB = MSUB_, NSUB = NSUB_, KB = KB_, NS = NS_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kRows = 32 * WM * MSUB, kCols = 32 * WN * NSUB;
  static constexpr int kA = kRows * KB, kB = kCols * KB, kStage = kA + kB, kRing = NS * kStage;
  static constexpr int kPer = 1024 / KB;  // rows per copy
  static constexpr int kACopies = kRows / kPer / kWaves, kBCopies = kCols / kPer / kWaves;
  static constexpr int kCopies = kACopies + kBCopies;  // per wave and group
  static constexpr int kSteps = KB / 32;
  static_assert(kRows % (kPer * kWaves) == 0 && kCols % (kPer * kWaves) == 0, "whole copies");

  struct Ctx {
    const char* x[kACopies];  // the lane's unit of each copy's row
    const char* w;            // the unit's columns
    uint32_t woff[kBCopies];
    int unit;  // the lane's unit within a group (the rows of its copies swizzle alike)
    uint32_t lds;
    int wave, lane, units;
  };
  struct Frag {
    i32x4_t a[MSUB], b[NSUB];
  };

  // Copy d of group g, of the wave's kCopies.
  static __device__ __forceinline__ void copy(const Ctx& c, int g, int stage, int d) {
    const uint32_t st = c.lds + stage * kStage;
    const bool in = g * (KB / 16) + c.unit < c.units;
    const bool whole = (g + 1) * (KB / 16) <= c.units;
    if (d < kACopies) {
      const char* p = c.x[d] + (size_t)g * KB;
      qmoe_gemm::dma16(whole || in ? p : reinterpret_cast<const char*>(zero_unit), st + (d * kWaves + c.wave) * 1024);
    } else {
      const int b = d - kACopies;
      const uint32_t dst = st + kA + (b * kWaves + c.wave) * 1024;
      if (whole) {
        qmoe_gemm::dma16s(c.w + (size_t)g * KB, c.woff[b], dst);
      } else {
        const char* p = c.w + (size_t)g * KB + c.woff[b];
        qmoe_gemm::dma16(in ? p : reinterpret_cast<const char*>(zero_unit), dst);
      }
    }
  }
  static __device__ __forceinline__ void read(const Ctx& c, const char* st, int kk, int row0, int col0, Frag& f) {
    const int l32 = c.lane % 32, unit = (2 * kk + c.lane / 32) ^ swz<KB>(l32);  // swz repeats every 16 rows
#pragma unroll
    for (int i = 0; i < MSUB; ++i)
      f.a[i] = *reinterpret_cast<const i32x4_t*>(st + (row0 + 32 * i + l32) * KB + unit * 16);
#pragma unroll
    for (int j = 0; j < NSUB; ++j)
      f.b[j] = *reinterpret_cast<const i32x4_t*>(st + kA + (col0 + 32 * j + l32) * KB + unit * 16);
  }
  // A step's products with PIECES calls of more(i) spread between them.
  template <int PIECES, class More>
  static __device__ __forceinline__ void products(const Frag& f, i32x16_t (&acc)[MSUB][NSUB], More more) {
#pragma unroll
    for (int j = 0; j < NSUB; ++j)
#pragma unroll
      for (int i = 0; i < MSUB; ++i) {
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.b[j], f.a[i], acc[i][j], 0, 0, 0);
        if constexpr (PIECES > 0) {
#pragma unroll
          for (int p = 0; p < PIECES; ++p)
            if (p * MSUB * NSUB / PIECES == j * MSUB + i) more(p);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
  }

  static __device__ __forceinline__ void run(const Product& a, const Unit& u, char* smem, float* sx, float* sw) {
    Ctx c;
    const int tid = fresh_tid();
    c.lane = tid % 64;
    c.wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = c.wave / WN, wn = c.wave % WN;
    c.units = (int)(a.K / 16);
    c.lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)smem);
    constexpr int kUnits = KB / 16;
    // a wave's copies are kWaves * kPer rows apart, a multiple of 16: their swizzle is one
    static_assert(kWaves * kPer % 16 == 0, "the copies' rows swizzle alike");
    c.unit = (c.lane % kUnits) ^ swz<KB>(c.wave * kPer + c.lane / kUnits);
#pragma unroll
    for (int d = 0; d < kACopies; ++d) {
      const int row = (d * kWaves + c.wave) * kPer + c.lane / kUnits;
      c.x[d] = reinterpret_cast<const char*>(a.x) + row_of(a, u, row) * a.K + c.unit * 16;
    }
    const int64_t n0 = (int64_t)u.e * a.N + u.o0;
    const int cols = (int)min((int64_t)kCols, a.N - u.o0);
    c.w = reinterpret_cast<const char*>(a.w) + qmoe_gemm::uniform64(n0 * a.K);
#pragma unroll
    for (int d = 0; d < kBCopies; ++d)
      c.woff[d] = (uint32_t)(min((d * kWaves + c.wave) * kPer + c.lane / kUnits, cols - 1) * (int)a.K + c.unit * 16);
    const int G = (c.units + kUnits - 1) / kUnits;
    const int row0 = 32 * MSUB * wm, col0 = 32 * NSUB * wn;

    // the scales, the rows' and the columns', into LDS ahead of everything else
    const uint32_t lsx = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)sx);
    const uint32_t lsw = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)sw);
    for (int i = c.wave * 64; i < kRows; i += kThreads) qmoe_gemm::dma4(a.sx + row_of(a, u, i + c.lane), lsx + i * 4);
    for (int i = c.wave * 64; i < kCols; i += kThreads) qmoe_gemm::dma4(a.sw + n0 + min(i + c.lane, cols - 1), lsw + i * 4);

    i32x16_t acc[MSUB][NSUB] = {};
    // past the end: the last group again, into stages that nothing reads any more
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
#pragma unroll
      for (int d = 0; d < kCopies; ++d) copy(c, min(i, G - 1), i, d);
    qmoe_gemm::wait_vmem<(NS - 2) * kCopies>();
    __builtin_amdgcn_s_barrier();
    Frag f[2];
    read(c, smem, 0, row0, col0, f[0]);
    int at = 0;  // the stage of group g
    for (int g = 0; g < G; ++g) {
      const char* st = smem + at * kStage;
      const int freed = at == 0 ? NS - 1 : at - 1, from = min(g + NS - 1, G - 1);
#pragma unroll
      for (int kk = 0; kk + 1 < kSteps; ++kk) {
        read(c, st, kk + 1, row0, col0, f[(kk + 1) & 1]);
        if (kk == 0) products<kCopies>(f[0], acc, [&](int p) { copy(c, from, freed, p); });
        else products<0>(f[kk & 1], acc, [](int) {});
        __builtin_amdgcn_sched_barrier(0);
      }
      at = at + 1 == NS ? 0 : at + 1;
      if (g + 1 < G) {
        // the next group landed (copies of NS - 2 groups after it may be in flight); this one's reads are done
        qmoe_gemm::wait_vmem<(NS - 2) * kCopies>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        read(c, smem + at * kStage, 0, row0, col0, f[kSteps & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
      products<0>(f[(kSteps - 1) & 1], acc, [](int) {});
      __builtin_amdgcn_sched_barrier(0);
    }
    qmoe_gemm::wait_vmem<0>();
    store(a, u, smem, sx, sw, acc);
  }

  // The results through LDS, a row subtile of every wave at a time, so that rows leave in whole lines.
  static __device__ __forceinline__ void store(const Product& a, const Unit& u, char* smem, const float* sx,
                                               const float* sw, i32x16_t (&acc)[MSUB][NSUB]) {
    const int tid = fresh_tid(), lane = tid % 64, l32 = lane % 32, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), wm = wave / WN, wn = wave % WN;
    const int size = a.dtype == QMOE_FP32 ? 4 : 2;
    const int64_t left = a.N - u.o0;
#pragma unroll
    for (int i = 0; i < MSUB; ++i) {
      __syncthreads();
      const int lr = 32 * wm + l32;
      const float s1 = sx[32 * MSUB * wm + 32 * i + l32];
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const int gi = (32 * NSUB * wn + 32 * j + 2 * v + 4 * h) / 4;  // four outputs
          const f32x4_t s = *reinterpret_cast<const f32x4_t*>(sw + 4 * gi);
          f32x4_t y;
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = scaled(acc[i][j][v + k], s1, s[k]);
          if (size == 4) {
            *reinterpret_cast<f32x4_t*>(smem + lr * (kCols * 4) + (gi ^ l32) * 16) = y;
          } else {
            uint2 o;
            if (a.dtype == QMOE_BF16) {
              o = make_uint2(qmoe_gemm::cvt_pk_bf16(y[0], y[1]), qmoe_gemm::cvt_pk_bf16(y[2], y[3]));
            } else {
              typedef _Float16 h4 __attribute__((ext_vector_type(4)));
              o = __builtin_bit_cast(uint2, h4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]});
            }
            *reinterpret_cast<uint2*>(smem + lr * (kCols * 2) + (gi ^ (2 * l32)) * 8) = o;
          }
        }
      __syncthreads();
      const int per = 16 / size, row_units = kCols / per;  // outputs of a 16-byte unit; units of a row
      for (int t = tid; t < 32 * WM * row_units; t += kThreads) {
        const int r = t / row_units, unit = t % row_units;
        const int row = 32 * MSUB * (r / 32) + 32 * i + r % 32;
        const int64_t n = per * unit;
        if (row >= u.valid || n >= left) continue;
        const int at = size == 4 ? (unit ^ (r % 32)) * 16 : ((2 * unit) ^ (2 * (r % 32))) * 8;
        const char* from = smem + r * (kCols * size) + at;
        char* to = static_cast<char*>(a.out) + ((u.row0 + row) * a.N + u.o0 + n) * size;
        const i32x4_t v = *reinterpret_cast<const i32x4_t*>(from);
        if (a.N % per == 0) {
          __builtin_nontemporal_store(v, reinterpret_cast<i32x4_t*>(to));
        } else if (n + per <= left) {
          reinterpret_cast<Loose16*>(to)->v = v;
        } else {
          for (int k = 0; k < left - n; ++k) {
            if (size == 4) reinterpret_cast<int*>(to)[k] = reinterpret_cast<const int*>(from)[k];
            else reinterpret_cast<uint16_t*>(to)[k] = reinterpret_cast<const uint16_t*>(from)[k];
          }
        }
      }
    }
  }
};

// The forms of a unit by its rows, widest first, each for units of more rows than the next takes.
template <class... Forms>
struct Pick;
template <class F>
struct Pick<F> {
  static constexpr int kRing = F::kRing, kStaged = 32 * F::WM * F::kCols * 4;
  static __device__ __forceinline__ void run(const Product& a, const Unit& u, char* smem, float* sx, float* sw) {
    F::run(a, u, smem, sx, sw);
  }
};
template <class F, class G, class... Rest>
struct Pick<F, G, Rest...> {
  typedef Pick<G, Rest...> Next;
  static constexpr int kRing = F::kRing > Next::kRing ? F::kRing : Next::kRing;
  static constexpr int kStaged = Pick<F>::kStaged > Next::kStaged ? Pick<F>::kStaged : Next::kStaged;
  static __device__ __forceinline__ void run(const Product& a, const Unit& u, char* smem, float* sx, float* sw) {
    if (u.valid > G::kRows) F::run(a, u, smem, sx, sw);
    else Next::run(a, u, smem, sx, sw);
  }
};

// ROWS: rows of a unit; BLOCKS per CU.
template <class Forms, int ROWS, int COLS, int BLOCKS>
__global__ __launch_bounds__(256, BLOCKS) void int8_gemm_kernel(Product a, int64_t row_units, int NB) {
  constexpr int kSmem = Forms::kRing > Forms::kStaged ? Forms::kRing : Forms::kStaged;
  constexpr bool kTable = ROWS == kTileRows;  // a tile table's units are its tiles
  constexpr int kOrder = kTable ? qmoe_gemm::kMaxOrder : 1;
  static_assert(BLOCKS * (kSmem + 4 * (ROWS + COLS + kOrder)) <= kLdsCU, "LDS per CU");
  __shared__ __attribute__((aligned(16))) char smem[kSmem];
  __shared__ __attribute__((aligned(16))) float sx[ROWS], sw[COLS];
  __shared__ int order[kOrder];
  const qmoe_gemm::Tiles table{a.offsets, a.tile_row, a.tile_exp, a.ntiles, a.n_rows, a.num_experts};
  bool ranked = false;
  if (kTable && a.offsets) {
    row_units = max(a.ntiles[0], 0);
    ranked = row_units <= kOrder;
    if (ranked) qmoe_gemm::rank_tiles(table, (int)row_units, order, reinterpret_cast<int*>(smem));
  }
  const qmoe_gemm::Snake snake(row_units * NB);
  constexpr int kBand = 2048 / COLS;  // column blocks of a band
  for (int64_t k = 0;; ++k) {
    const int64_t at = snake.unit(k);
    if (at < 0) break;
    Unit u;
    int col;
    if (kTable && a.offsets) {
      const int64_t tile = at / NB;
      col = (int)(at % NB);
      const qmoe_gemm::TileRows t = qmoe_gemm::tile_rows_of(table, ranked ? order[tile] : (int)tile);
      u.e = __builtin_amdgcn_readfirstlane(t.e);
      u.valid = __builtin_amdgcn_readfirstlane(t.valid);
      u.row0 = qmoe_gemm::uniform64(t.row0);
    } else {
      const int64_t band = at / (row_units * kBand), in = at % (row_units * kBand);
      const int wide = (int)min((int64_t)kBand, NB - band * kBand);
      col = (int)(band * kBand + in % wide);
      u.e = 0;
      u.row0 = in / wide * ROWS;
      u.valid = (int)min((int64_t)ROWS, a.n_rows - u.row0);
    }
    if (u.valid <= 0) continue;
    u.o0 = (int64_t)__builtin_amdgcn_readfirstlane(col) * COLS;
    Forms::run(a, u, smem, sx, sw);
    __syncthreads();  // the ring and the scales are free for the next unit
  }
}

// 256 x 256 outputs, one block per CU; 128 x 256, two, with shorter forms for the ends of segments.
typedef Pick<Form<2, 2, 4, 4, 128, 2>> Wide;
typedef Pick<Form<2, 2, 2, 4, 64, 3>, Form<1, 4, 2, 2, 64, 3>> Tile;

template <class Forms, int ROWS, int BLOCKS>
void launch(const Product& a, int64_t max_tiles, hipStream_t st) {
  const int64_t NB = (a.N + 255) / 256, rows = a.offsets ? max_tiles : (a.n_rows + ROWS - 1) / ROWS;
  const dim3 grid((unsigned)qmoe_gemm::grid_blocks(rows * NB, BLOCKS));
  int8_gemm_kernel<Forms, ROWS, 256, BLOCKS><<<grid, dim3(256), 0, st>>>(a, rows, (int)NB);
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
  hipStream_t st = qmoe::as_stream(stream);
  const int64_t wide = (n_rows + 255) / 256 * ((N + 255) / 256);
  if (!any && wide >= 192) launch<Wide, 256, 1>(a, max_tiles, st);
  else launch<Tile, kTileRows, 2>(a, max_tiles, st);
  return qmoe::launch_status("int8_gemm_kernel");
}
