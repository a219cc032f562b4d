// Products of mxfp4 weights with many rows on the matrix cores: bf16
// activations either way round (x W^T over the packed axis, x W over the
// rows), and activations in mxfp4 too (format in mxfp4.h).  Rows are those of
// a tile table (sorted by expert), or of one expert without a table.
#include <algorithm>
#include <type_traits>

#include "gemm_common.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"

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
  // kQQ: scales in lines (mxfp4.h), null: as they are in s and xs
  const uint32_t *sl, *xl;
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

// Layout of the work.  A unit is a tile of up to 128 rows of one expert times
// 256 outputs.  Four waves share it two by two: wave (wm, wn) takes half the
// tile's rows and 128 of the outputs, so weights are converted twice per tile
// and activations read twice from LDS (one by four would halve the first and
// double the second, and LDS reads are the scarcer: at 128 B a clock and CU
// they take 55% of the matrix cores' time as it is; measured, either way takes
// 61 us for 4096 x 2048 x 4096).  Blocks are persistent, two per CU, and take
// the units heavy-first (gemm_common.h).  Shorter tiles run in forms of 32, 64
// and 96 rows (the last up to 128 in steps of 32; both mxfp4: 64 and 128): with
// 64 and 128 alone 40,960 rows of 256 experts pay for 20% more rows than they
// have, with these for 10%.
//
// What bounds it: a product of 68.7 GFLOP takes 61 us (1.1 PFLOP/s) forward, at
// the card's power limit (a loop of nothing but these instructions runs at 1.8
// GHz of 2.4).  Transposed it takes 72 to 80 back to back (82 to 90 where each
// is waited for): for the same products it issues twice the matrix
// instructions, and a permute besides each conversion; blocks alone on their
// CU are as fast as two, copies five groups ahead as fast as three.  4096^3 in
// mxfp4 takes 49 us (2.8 PFLOP/s), bound by the copies into LDS.
//
// Operands reach LDS by asynchronous copies into a ring of NS stages and are
// read from there as matrix fragments; the fragments of a step are prepared
// during the step before.  The barrier that hands over a stage stands before
// a group's last step, whose operands are in registers by then: past it the
// next group's first fragments are read, and the stage just emptied takes the
// copies of NS groups ahead.
//
// Where the units are too few for that to fill the chip (SPLIT), a unit is 64
// (32) rows times 128 outputs, every wave computes all of it over a quarter of
// the contraction, in a ring of its own without barriers, and the four partial
// sums are added through LDS in wave order: an eighth of the work per unit.
constexpr int kRowsHalf = kTileRows / 2;
constexpr int kWideCols = 256, kSplitCols = 128;
constexpr int kLdsCU = 160 * 1024;
__device__ __attribute__((aligned(16))) uint32_t zero_page[4];  // what copies past the contraction's end read

__device__ __forceinline__ void dma1s(const void* sbase, uint32_t voff, uint32_t lds_base) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_ubyte %1, %2"
      :
      : "s"(lds_base), "v"(voff), "s"(sbase)
      : "memory", "m0");
}
__device__ __forceinline__ void dma1(const void* g, uint32_t lds_base) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_ubyte %1, off"
      :
      : "s"(lds_base), "v"(g)
      : "memory", "m0");
}

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

// What differs between the two ways: outputs per unit, the waves that fill one
// ring, and the wave's part of the groups (in steps of UNIT groups).
template <bool SPLIT>
struct Geo {
  static constexpr int kCols = SPLIT ? kSplitCols : kWideCols;
  static constexpr int kWaves = SPLIT ? 1 : 4;  // per ring
  static constexpr int kRings = SPLIT ? 4 : 1;
  static __device__ __forceinline__ void barrier() {
    if constexpr (!SPLIT) __builtin_amdgcn_s_barrier();
  }
  template <int UNIT>
  static __device__ __forceinline__ void part(int groups, int wave, int* first, int* end) {
    if constexpr (SPLIT) {
      const int per = ((groups + UNIT - 1) / UNIT + 3) / 4 * UNIT;
      *first = min(wave * per, groups);
      *end = min(*first + per, groups);
    } else {
      *first = 0;
      *end = groups;
    }
  }
};

// Swizzle of the eight 16-byte units of a 128-byte activation row in LDS, of
// the four of a 64-byte row: conflict-free 16-byte reads of one unit by
// sixteen consecutive rows.
__device__ __forceinline__ int swz8(int row) { return (row & 7) ^ ((row >> 3) & 1); }
__device__ __forceinline__ int swz4(int row) { return (row >> 2) & 3; }

// Sources of the copies of the tile's activation rows: copy d of a wave fills
// 1 KiB, 64 / UNITS rows of UNITS 16-byte units.  Rows past the tile's end are
// its last row again (nothing of them is stored).
template <int COPIES, int UNITS, int WAVES>
struct RowSrc {
  const char* p[COPIES];
  int unit0;
  // source unit of copy d: the row's swizzle differs between copies only where a lone wave makes all of them
  __device__ __forceinline__ int unit(int d) const { return UNITS == 8 && WAVES == 1 ? unit0 ^ (d & 1) : unit0; }
};
template <int COPIES, int UNITS, int WAVES>
__device__ __forceinline__ RowSrc<COPIES, UNITS, WAVES> row_sources(const GemmArgs& a, const Unit& u, const void* base,
                                                             int64_t pitch, int wave, int lane) {
  RowSrc<COPIES, UNITS, WAVES> r;
  r.unit0 = (lane % UNITS) ^ (UNITS == 8 ? swz8(wave * 8 + lane / UNITS) : swz4(lane / UNITS));
#pragma unroll
  for (int d = 0; d < COPIES; ++d) {
    const int row = (d * WAVES + wave) * (64 / UNITS) + lane / UNITS;
    const int64_t i = u.row0 + min(row, u.valid - 1);
    const int64_t x = min(max(a.x_rows ? (int64_t)a.x_rows[i] : i, (int64_t)0), a.n_x - 1);
    r.p[d] = static_cast<const char*>(base) + x * pitch + r.unit(d) * 16;
  }
  return r;
}

// One pass of a unit's results, staged in LDS as 64 rows of 256 bf16, so that a
// row leaves as 512 contiguous bytes.  HALF rows per wave: with two waves along
// the rows (WM) a pass takes 32 of each one's, else 64 of the one's.
template <int WM, int HALF>
__device__ __forceinline__ void store_rows(const GemmArgs& a, const char* ep, const Unit& u, int64_t O, int pass) {
  uint16_t* out = static_cast<uint16_t*>(a.out);
  const int tid = fresh_tid();
  const auto row_of = [&](int lr) {  // past the tile's end: not stored
    if constexpr (WM == 1) return 64 * pass + lr;
    const int r = 32 * pass + lr % 32;
    return r < HALF ? HALF * (lr / 32) + r : kTileRows;
  };
  if (O % 8 == 0) {
    for (int i = tid; i < 64 * 32; i += 256) {
      const int lr = i / 32, unit = i % 32;
      const int row = row_of(lr);
      if (row < u.valid && u.o0 + 8 * unit < O)
        __builtin_nontemporal_store(
            *reinterpret_cast<const i32x4_t*>(ep + lr * 512 + ((2 * unit) ^ (2 * (lr % 32))) * 8),
            reinterpret_cast<i32x4_t*>(out + (u.row0 + row) * O + u.o0 + 8 * unit));
    }
  } else {
    for (int i = tid; i < 64 * 256; i += 256) {
      const int lr = i / 256, c = i % 256;
      const int row = row_of(lr);
      if (row < u.valid && u.o0 + c < O)
        out[(u.row0 + row) * O + u.o0 + c] =
            *reinterpret_cast<const uint16_t*>(ep + lr * 512 + ((c / 4) ^ (2 * (lr % 32))) * 8 + (c % 4) * 2);
    }
  }
}

// A split unit's results: the waves' partial sums, staged as ROWS x 128 floats
// each, 16-byte units of a row swizzled by row, added in wave order.
__device__ __forceinline__ int part_at(int row, int col4) { return (row * 32 + (col4 ^ (row & 31))) * 16; }
template <int ROWS>
__device__ __forceinline__ void store_parts(const GemmArgs& a, const char* ep, const Unit& u, int64_t O) {
  const int tid = fresh_tid();
  for (int i = tid; i < ROWS * 32; i += 256) {
    const int row = i / 32, c = i % 32;
    if (row >= u.valid) continue;
    f32x4_t v = *reinterpret_cast<const f32x4_t*>(ep + part_at(row, c));
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const f32x4_t p = *reinterpret_cast<const f32x4_t*>(ep + w * ROWS * 512 + part_at(row, c));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += p[k];
    }
    const int64_t o = u.o0 + 4 * c, at = (u.row0 + row) * O + o;
    if (o >= O) continue;
    if (a.out_f32) {
      float* out = static_cast<float*>(a.out) + at;
      if (O % 4 == 0) *reinterpret_cast<f32x4_t*>(out) = v;
      else
        for (int k = 0; k < 4 && o + k < O; ++k) out[k] = v[k];
    } else {
      uint16_t* out = static_cast<uint16_t*>(a.out) + at;
      const uint2 b = make_uint2(qmoe_gemm::cvt_pk_bf16(v[0], v[1]), qmoe_gemm::cvt_pk_bf16(v[2], v[3]));
      if (O % 4 == 0) *reinterpret_cast<uint2*>(out) = b;
      else
        for (int k = 0; k < 4 && o + k < O; ++k) out[k] = (uint16_t)((k < 2 ? b.x : b.y) >> (16 * (k & 1)));
    }
  }
}

// ----------------------------------------------------------- x W^T, bf16 x
//
// Contraction in groups of 64, weights in pairs of groups, so that a weight
// row is copied 64 bytes at a time.  Per group a wave reads each of its four
// 32-column subtiles' codes once (16 bytes, one block, per lane) and converts
// a word of each per step: lane half h supplies elements 32h + 8kk .. + 7 of
// the group at step kk, from word kk of its block.
// WM: waves along the rows, of four.  S4: scales copied four blocks at a time (K % 128 == 0, aligned)
template <bool S4, int WM, int MSUB, bool SPLIT>
struct Fwd {
  typedef Geo<SPLIT> Way;
  static constexpr int kCols = Way::kCols, kRows = 32 * WM * MSUB;
  static constexpr int NSUB = SPLIT ? 4 : 2 * WM;  // 32-column subtiles per wave
  static constexpr int kA = kRows * 128, kB = kCols * 64, kS = kCols * (S4 ? 4 : 16);
  static constexpr int kBOff = 2 * kA, kSOff = kBOff + 2 * kB;
  static constexpr int kRing = kSOff + 2 * kS;
  static constexpr int kACopies = kRows / 8 / Way::kWaves, kBCopies = kCols / 16 / Way::kWaves;
  static constexpr int kSCopies = kCols / 64 / Way::kWaves;

  struct Ctx {
    RowSrc<kACopies, 8, Way::kWaves> x;
    const char *w, *s;  // the column block's codes and scales
    uint32_t woff[kBCopies];  // copy d's column and unit; the unit
    uint32_t soff[kSCopies];
    int wunit;
    uint32_t lds;
    int wave, lane, units;  // wave: of those that fill the ring
    int64_t C;
  };

  static __device__ __forceinline__ void copy_x(const Ctx& c, int g, int stage) {
    const uint32_t dst = c.lds + stage * kA + c.wave * 1024;
    const bool whole = (int64_t)(g + 1) * 64 <= c.C;
    if (whole) {
#pragma unroll
      for (int d = 0; d < kACopies; ++d) qmoe_gemm::dma16(c.x.p[d] + (size_t)g * 128, dst + d * Way::kWaves * 1024);
    } else {
#pragma unroll
      for (int d = 0; d < kACopies; ++d) {
        const bool in = (int64_t)g * 64 + c.x.unit(d) * 8 < c.C;
        qmoe_gemm::dma16(in ? c.x.p[d] + (size_t)g * 128 : reinterpret_cast<const char*>(zero_page),
                         dst + d * Way::kWaves * 1024);
      }
    }
  }
  static __device__ __forceinline__ void copy_w(const Ctx& c, int p, int stage) {
    const uint32_t dst = c.lds + kBOff + stage * kB + c.wave * 1024;
    const uint32_t sdst = c.lds + kSOff + stage * kS + c.wave * 256;
    const bool whole = 4 * (p + 1) <= c.units;
#pragma unroll
    for (int d = 0; d < kBCopies; ++d) {
      if (whole) {
        qmoe_gemm::dma16s(c.w + (size_t)p * 64, c.woff[d], dst + d * Way::kWaves * 1024);
      } else {
        const char* q = c.w + (size_t)p * 64 + c.woff[d];
        if (4 * p + c.wunit >= c.units) q = reinterpret_cast<const char*>(zero_page);
        qmoe_gemm::dma16(q, dst + d * Way::kWaves * 1024);
      }
    }
#pragma unroll
    for (int d = 0; d < kSCopies; ++d) {
      if constexpr (S4) {
        qmoe_gemm::dma4s(c.s + (size_t)p * 4, c.soff[d], sdst + d * 256);
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (4 * p + b < c.units) dma1s(c.s + (size_t)p * 4 + b, c.soff[d], sdst + b * kCols * 4 + d * 256);
          else dma1(zero_page, sdst + b * kCols * 4 + d * 256);
        }
      }
    }
  }

  struct Frag {
    i32x4_t a[MSUB], b[NSUB];
  };
  struct Codes {
    i32x4_t w[NSUB];
    float s[NSUB];
  };
  // Group `at` of the wave's part (its stages, and the half of its pair): a constant in the main loop.
  static __device__ __forceinline__ void read_x(const Ctx& c, const char* smem, int at, int kk, int row0, Frag& f) {
    const int l32 = c.lane % 32, h = c.lane / 32;
    const char* st = smem + row0 * 128 + l32 * 128 + ((4 * h + kk) ^ swz8(l32)) * 16 + (at & 1) * kA;
#pragma unroll
    for (int i = 0; i < MSUB; ++i)  // swz8(row0 + 32 i + l32) == swz8(l32)
      f.a[i] = *reinterpret_cast<const i32x4_t*>(st + i * 4096);
  }
  static __device__ __forceinline__ Codes read_codes(const Ctx& c, const char* smem, int at, int col0) {
    const int l32 = c.lane % 32, h = c.lane / 32, half = at & 1, stage = (at >> 1) & 1;
    // the lane's unit 2 half + h, swizzled: swz4(col) == swz4(l32)
    const char* st = smem + kBOff + (col0 + l32) * 64 + ((h ^ swz4(l32)) ^ (2 * half)) * 16 + stage * kB;
    const char* ss = smem + kSOff + (col0 + l32 + (S4 ? 0 : h * kCols)) * 4 + stage * kS + (S4 ? 0 : half * 2 * kCols * 4);
    Codes r;
#pragma unroll
    for (int j = 0; j < NSUB; ++j) {
      r.w[j] = *reinterpret_cast<const i32x4_t*>(st + j * 2048);
      const uint32_t v = *reinterpret_cast<const uint32_t*>(ss + j * 128);
      r.s[j] = S4 ? scale_of(v, 2 * half + h) : scale_of(v);
    }
    return r;
  }
  static __device__ __forceinline__ void convert(const Codes& q, int kk, int j, Frag& f) {
    uint32_t o[4];
    unpack8((uint32_t)q.w[j][kk], q.s[j], o);
#pragma unroll
    for (int d = 0; d < 4; ++d) f.b[j][d] = (int)o[d];
  }
  // One step's products, the next step's conversions between them.
  template <bool NEXT>
  static __device__ __forceinline__ void step(const Frag& cur, Frag& nxt, const Codes& q, int kkn,
                                              f32x16_t (&acc)[MSUB][NSUB]) {
#pragma unroll
    for (int j = 0; j < NSUB; ++j) {
#pragma unroll
      for (int i = 0; i < MSUB; ++i) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, cur.b[j]),
                                                            __builtin_bit_cast(bf16x8_t, cur.a[i]), acc[i][j], 0, 0, 0);
        if constexpr (NEXT) {
          if (i == 0) convert(q, kkn, j, nxt);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // A split wave's partial sums into LDS (part_at's layout), once no wave reads its ring any more.
  static __device__ __forceinline__ void put_parts(char* ep, int l32, int h, const f32x16_t (&acc)[MSUB][NSUB]) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MSUB; ++i)
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *reinterpret_cast<f32x4_t*>(ep + part_at(32 * i + l32, (32 * j + 2 * v + 4 * h) / 4)) =
              f32x4_t{acc[i][j][v], acc[i][j][v + 1], acc[i][j][v + 2], acc[i][j][v + 3]};
  }

  static __device__ __forceinline__ void run(const GemmArgs& a, const Unit& u, char* block_smem) {
    Ctx c;
    const int tid = fresh_tid();
    c.lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = SPLIT || WM == 1 ? 0 : wave / 2, wn = SPLIT ? 0 : WM == 1 ? wave : wave % 2;
    char* smem = block_smem + (SPLIT ? wave * kRing : 0);
    c.wave = SPLIT ? 0 : wave;
    c.units = (int)(a.K / kBlock);
    c.C = a.K;
    c.lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)smem);
    c.x = row_sources<kACopies, 8, Way::kWaves>(a, u, a.x, a.ldx * 2, c.wave, c.lane);
    const int64_t row = (int64_t)u.e * a.N + u.o0;
    const int cols = (int)min((int64_t)kCols, a.N - u.o0);
    c.w = reinterpret_cast<const char*>(a.w) + qmoe_gemm::uniform64(row * c.units * 16);
    c.s = reinterpret_cast<const char*>(a.s) + qmoe_gemm::uniform64(row * c.units);
    c.wunit = (c.lane % 4) ^ swz4(c.lane / 4);  // swz4 repeats every 16 columns
#pragma unroll
    for (int d = 0; d < kBCopies; ++d) {
      const int col = (d * Way::kWaves + c.wave) * 16 + c.lane / 4;
      c.woff[d] = (uint32_t)(min(col, cols - 1) * c.units * 16 + c.wunit * 16);
    }
#pragma unroll
    for (int d = 0; d < kSCopies; ++d)
      c.soff[d] = (uint32_t)(min((d * Way::kWaves + c.wave) * 64 + c.lane, cols - 1) * c.units);
    int g0, G;  // this wave's groups, whole pairs
    Way::template part<2>((int)((a.K + 63) / 64), wave, &g0, &G);
    const int P = (G + 1) / 2;
    const int row0 = 32 * MSUB * wm, col0 = 32 * NSUB * wn;

    f32x16_t acc[MSUB][NSUB] = {};
    if (!SPLIT || g0 < G) {
      constexpr int kPairCopies = kBCopies + kSCopies * (S4 ? 1 : 4);
      const int p0 = g0 / 2;
      copy_x(c, g0, 0);
      copy_w(c, p0, 0);
      if (g0 + 1 < G) copy_x(c, g0 + 1, 1);
      if (p0 + 1 < P) copy_w(c, p0 + 1, 1);
      if (p0 + 1 < P) qmoe_gemm::wait_vmem<kACopies + kPairCopies>();
      else qmoe_gemm::wait_vmem<0>();
      Way::barrier();
      Frag fa, fb;
      Codes q = read_codes(c, smem, 0, col0);
      read_x(c, smem, 0, 0, row0, fa);
#pragma unroll
      for (int j = 0; j < NSUB; ++j) convert(q, 0, j, fa);
      int g = g0;
      // a group but the last, `at` of the part (mod 4: a constant where four of them are run in turn)
      const auto group = [&](auto at_) {
        const int at = at_ & 3;
        read_x(c, smem, at, 1, row0, fb);
        step<true>(fa, fb, q, 1, acc);
        read_x(c, smem, at, 2, row0, fa);
        step<true>(fb, fa, q, 2, acc);
        read_x(c, smem, at, 3, row0, fb);
        step<true>(fa, fb, q, 3, acc);
        // the next group landed, a pair of weights behind it may be in flight; this one's stages are read
        if (at % 2 == 0 && g / 2 + 1 < P) qmoe_gemm::wait_vmem<kPairCopies>();
        else qmoe_gemm::wait_vmem<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        Way::barrier();
        if (g + 2 < G) copy_x(c, g + 2, at % 2);
        if (at % 2 && g / 2 + 2 < P) copy_w(c, g / 2 + 2, at / 2);
        q = read_codes(c, smem, (at + 1) % 4, col0);
        read_x(c, smem, (at + 1) % 4, 0, row0, fa);
        step<true>(fb, fa, q, 0, acc);
        ++g;
      };
      while (g + 4 < G) {
        group(std::integral_constant<int, 0>{});
        group(std::integral_constant<int, 1>{});
        group(std::integral_constant<int, 2>{});
        group(std::integral_constant<int, 3>{});
      }
      while (g + 1 < G) group(g - g0);
      const int at = (G - 1 - g0) & 3;
      read_x(c, smem, at, 1, row0, fb);
      step<true>(fa, fb, q, 1, acc);
      read_x(c, smem, at, 2, row0, fa);
      step<true>(fb, fa, q, 2, acc);
      read_x(c, smem, at, 3, row0, fb);
      step<true>(fa, fb, q, 3, acc);
      step<false>(fb, fa, q, 0, acc);
    }
    const int lane = fresh_tid() % 64, l32 = lane % 32, h = lane / 32;
    if constexpr (SPLIT) {
      put_parts(block_smem + wave * kRows * 512, l32, h, acc);
      __syncthreads();
      store_parts<kRows>(a, block_smem, u, a.N);
      return;
    }
    if (a.out_f32) {
#pragma unroll
      for (int i = 0; i < MSUB; ++i) {
        const int r = row0 + 32 * i + l32;
        if (r >= u.valid) continue;
#pragma unroll
        for (int j = 0; j < NSUB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int64_t o = u.o0 + col0 + 32 * j + 8 * (v / 4) + 4 * h + v % 4;
            if (o < a.N) static_cast<float*>(a.out)[(u.row0 + r) * a.N + o] = acc[i][j][v];
          }
      }
      return;
    }
    constexpr int kPer = WM == 1 ? 2 : 1;  // row subtiles per pass
#pragma unroll
    for (int i = 0; i < MSUB; ++i) {
      if (i % kPer == 0) __syncthreads();
      const int lr = 32 * (WM == 1 ? i % 2 : wm) + l32;
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const int gi = (col0 + 32 * j + 2 * v + 4 * h) / 4;
          *reinterpret_cast<uint2*>(smem + lr * 512 + (gi ^ (2 * l32)) * 8) =
              make_uint2(qmoe_gemm::cvt_pk_bf16(acc[i][j][v], acc[i][j][v + 1]),
                         qmoe_gemm::cvt_pk_bf16(acc[i][j][v + 2], acc[i][j][v + 3]));
        }
      if (i % kPer == kPer - 1 || i == MSUB - 1) {
        __syncthreads();
        store_rows<WM, 32 * MSUB>(a, smem, u, a.N, i / kPer);
      }
    }
  }
};

// ------------------------------------------------------------- x W, bf16 x
//
// The contraction runs over the weights' rows n, in groups of 64; the outputs
// lie along the packed axis.  A lane takes one word of codes (eight outputs)
// of eight consecutive rows n: four conversions a word give pairs of outputs
// of one n, and a byte permute of two n's words gives the pairs of n of one
// output that the matrix instruction wants.  With v_mfma_f32_16x16x32 the
// sixteen words of a wave's 128 outputs are the sixteen lanes of a quarter
// wave and the four quarters the four octets of n, so no value crosses lanes:
// the sixteen outputs of subtile j are 8c + j, c = 0 .. 15.  Eight conversions
// and eight permutes go with eight products of 64 rows, spread between them (in
// runs of their own: 1 to 2% slower).
template <bool S4, int MSUB, bool SPLIT>  // MSUB: 16-row subtiles per wave
struct Trn {
  typedef Geo<SPLIT> Way;
  static constexpr int kCols = Way::kCols, kRows = (SPLIT ? 16 : 32) * MSUB;
  static constexpr int kUnits = kCols / kBlock;  // 16-byte units of codes per row n
  static constexpr int kA = kRows * 128, kB = 64 * kUnits * 16, kS = 64 * kUnits * (S4 ? 1 : 4);
  static constexpr int kStage = kA + kB + kS;
  static constexpr int NS = 3;
  static constexpr int kRing = NS * kStage;
  static constexpr int kACopies = kRows / 8 / Way::kWaves;
  static constexpr int kBCopies = SPLIT ? 4 : 2;
  static constexpr int kSCopies = S4 ? 1 : SPLIT ? 4 : 2;
  static constexpr int kCopies = kACopies + kBCopies + kSCopies;  // per wave and group

  struct Ctx {
    RowSrc<kACopies, 8, Way::kWaves> x;
    const char *w, *s;  // of the expert's first row, at the column block
    int64_t wpitch, spitch;
    uint32_t woff[kBCopies], soff[kSCopies];  // the lane's bytes from there
    int pos;                                  // row slot of copy 0
    uint32_t lds;
    int wave, lane;  // wave: of those that fill the ring
    int64_t C;
    __device__ __forceinline__ int row(int d) const { return w_row(pos + (SPLIT ? 16 : 32) * d); }
  };

  static __device__ __forceinline__ void copy(const Ctx& c, int g) {
    const uint32_t st = c.lds + (g % NS) * kStage;
    const uint32_t xd = st + c.wave * 1024, wd = st + kA + c.wave * 1024, sd = st + kA + kB;
    const int64_t left = c.C - (int64_t)g * 64;  // rows n of this group and after
    const char* w = c.w + (int64_t)g * 64 * c.wpitch;
    const char* s = c.s + (int64_t)g * 64 * c.spitch;
    if (left >= 64) {
#pragma unroll
      for (int d = 0; d < kACopies; ++d) qmoe_gemm::dma16(c.x.p[d] + (size_t)g * 128, xd + d * Way::kWaves * 1024);
#pragma unroll
      for (int d = 0; d < kBCopies; ++d) qmoe_gemm::dma16s(w, c.woff[d], wd + d * Way::kWaves * 1024);
#pragma unroll
      for (int d = 0; d < kSCopies; ++d) {
        if constexpr (S4) qmoe_gemm::dma4s(s, c.soff[d], sd + (c.wave & 1) * 256);
        else dma1s(s, c.soff[d], sd + (kSCopies * c.wave + d) * 256);
      }
    } else {  // the last group of a contraction that is no multiple of 64
      const char* zero = reinterpret_cast<const char*>(zero_page);
#pragma unroll
      for (int d = 0; d < kACopies; ++d)
        qmoe_gemm::dma16(c.x.unit(d) * 8 < left ? c.x.p[d] + (size_t)g * 128 : zero, xd + d * Way::kWaves * 1024);
#pragma unroll
      for (int d = 0; d < kBCopies; ++d)
        qmoe_gemm::dma16(c.row(d) < left ? w + c.woff[d] : zero, wd + d * Way::kWaves * 1024);
#pragma unroll
      for (int d = 0; d < kSCopies; ++d) {
        const char* p = c.lane < left ? s + c.soff[d] : zero;
        if constexpr (S4) qmoe_gemm::dma4(p, sd + (c.wave & 1) * 256);
        else dma1(p, sd + (kSCopies * c.wave + d) * 256);
      }
    }
  }
  // Row n of the group in the codes' row slot `pos` (its own inverse), and the unit in a unit slot: chosen so that
  // the words that a wave reads at once, those of rows n + 8 q, fall on all banks, and those of half a wave on half.
  static __device__ __forceinline__ int w_row(int pos) {
    return SPLIT ? pos ^ ((pos >> 3) & 3) : pos ^ ((pos >> 4) & 1);
  }
  static __device__ __forceinline__ int w_unit(int slot, int pos) { return SPLIT ? slot : slot ^ (4 * ((pos >> 3) & 1)); }

  struct Words {
    uint32_t w[8];
    float s[8];
  };
  static __device__ __forceinline__ Words read_words(const Ctx& c, const char* smem, int g, int s, int wn) {
    const int co = c.lane % 16, q = c.lane / 16;
    const char* st = smem + (g % NS) * kStage + kA;
    const int unit = w_unit(4 * wn + co / 4, 8 * q);
    Words r;
    // w_row(8 q + i) = 8 q + (i & ~m) + w_row of the low bits: few bases, the rest in the offsets
    constexpr int m = SPLIT ? 3 : 1, kPitch = kUnits * 16;
    const char* base[m + 1];
#pragma unroll
    for (int i = 0; i <= m; ++i) base[i] = st + w_row(8 * q + i) * kPitch + unit * 16 + (co % 4) * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r.w[i] = *reinterpret_cast<const uint32_t*>(base[i & m] + (32 * s + (i & ~m)) * kPitch);
    const int blk = 4 * wn + co / 4;
    const char* ss = st + kB + (S4 ? wn : blk) * 256 + (32 * s + 8 * q) * 4;
    const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(ss), hi = *reinterpret_cast<const i32x4_t*>(ss + 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t v = (uint32_t)(i < 4 ? lo[i & 3] : hi[i & 3]);
      r.s[i] = S4 ? scale_of(v, co / 4) : scale_of(v);
    }
    return r;
  }
  // Four values of the fragments of outputs 8c + 2T and 8c + 2T + 1, those of rows n 2i and 2i + 1.
  template <int T>
  static __device__ __forceinline__ void pair(const Words& q, int i, i32x4_t (&b)[2]) {
    const uint32_t lo = pair_of<T>(q.w[2 * i], q.s[2 * i]), hi = pair_of<T>(q.w[2 * i + 1], q.s[2 * i + 1]);
    b[0][i] = (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
    b[1][i] = (int)__builtin_amdgcn_perm(hi, lo, 0x07060302u);
  }
  static __device__ __forceinline__ void read_x(const Ctx& c, const char* smem, int g, int s, int row0,
                                                i32x4_t (&f)[MSUB]) {
    const int l16 = c.lane % 16, q = c.lane / 16;
    const char* st = smem + (g % NS) * kStage + row0 * 128;
#pragma unroll
    for (int i = 0; i < MSUB; ++i)
      f[i] = *reinterpret_cast<const i32x4_t*>(st + (16 * i + l16) * 128 + ((4 * s + q) ^ swz8(l16)) * 16);
  }
  // The products of outputs 8c + 2t and 8c + 2t + 1, with `pieces` calls of more(i) spread between them.
  template <int PIECES, class More>
  static __device__ __forceinline__ void products(const i32x4_t (&x)[MSUB], const i32x4_t (&b)[2],
                                                  f32x4_t (&acc)[MSUB][8], int t, More more) {
#pragma unroll
    for (int m = 0; m < 2 * MSUB; ++m) {
      const int v = m / MSUB, i = m % MSUB;
      acc[i][2 * t + v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b[v]),
                                                                  __builtin_bit_cast(bf16x8_t, x[i]),
                                                                  acc[i][2 * t + v], 0, 0, 0);
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
        if (p * 2 * MSUB / PIECES == m) more(p);
      if (PIECES) __builtin_amdgcn_sched_barrier(0);
    }
  }
  // One step, its first outputs' fragments in b0: the others are prepared during the first half of its products, so
  // that the current words are used up when next() reads the next step's words and activations, and the next step's
  // first fragments, into b1, during the last quarter.
  template <class Next>
  static __device__ __forceinline__ void step(const i32x4_t (&x)[MSUB], Words& w, i32x4_t (&b0)[2], i32x4_t (&b1)[2],
                                              i32x4_t (&b2)[2], f32x4_t (&acc)[MSUB][8], Next next) {
    products<6>(x, b0, acc, 0, [&](int p) {
      if (p < 4) pair<1>(w, p, b1);
      else pair<2>(w, p - 4, b2);
    });
    products<6>(x, b1, acc, 1, [&](int p) {
      if (p < 2) pair<2>(w, p + 2, b2);
      else pair<3>(w, p - 2, b0);
    });
    next();
    products<0>(x, b2, acc, 2, [](int) {});
    __builtin_amdgcn_sched_barrier(0);
    products<4>(x, b0, acc, 3, [&](int p) { pair<0>(w, p, b1); });
  }

  static __device__ __forceinline__ void run(const GemmArgs& a, const Unit& u, char* block_smem) {
    Ctx c;
    const int tid = fresh_tid();
    c.lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = SPLIT ? 0 : wave / 2, wn = SPLIT ? 0 : wave % 2;
    char* smem = block_smem + (SPLIT ? wave * kRing : 0);
    c.wave = SPLIT ? 0 : wave;
    const int64_t units = a.K / kBlock;
    c.C = a.N;
    c.lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)smem);
    c.x = row_sources<kACopies, 8, Way::kWaves>(a, u, a.x, a.ldx * 2, c.wave, c.lane);
    const int64_t row = (int64_t)u.e * a.N, u0 = u.o0 / kBlock;
    const int last = (int)min((int64_t)kUnits, units - u0) - 1;  // columns past the end: the last again
    c.wpitch = units * 16;
    c.spitch = units;
    c.pos = c.wave * 8 + c.lane / kUnits;
    c.w = reinterpret_cast<const char*>(a.w) + qmoe_gemm::uniform64((row * units + u0) * 16);
    c.s = reinterpret_cast<const char*>(a.s) + qmoe_gemm::uniform64(row * units + u0);
    const int unit = min(w_unit(c.lane % kUnits, c.pos), last);
#pragma unroll
    for (int d = 0; d < kBCopies; ++d) c.woff[d] = (uint32_t)(c.row(d) * (int)c.wpitch + unit * 16);
#pragma unroll
    for (int d = 0; d < kSCopies; ++d) {
      const int blk = S4 ? (SPLIT ? 0 : 4 * (c.wave & 1)) : kSCopies * c.wave + d;
      c.soff[d] = (uint32_t)(c.lane * (int)c.spitch + (blk <= last ? blk : S4 ? 0 : last));
    }
    int g0, G;  // this wave's groups
    Way::template part<1>((int)((a.N + 63) / 64), wave, &g0, &G);
    const int row0 = 16 * MSUB * wm;

    f32x4_t acc[MSUB][8] = {};
    if (!SPLIT || g0 < G) {
#pragma unroll
    for (int i = 0; i < NS; ++i) copy(c, min(g0 + i, G - 1));
    qmoe_gemm::wait_vmem<(NS - 1) * kCopies>();
    Way::barrier();
    i32x4_t xa[MSUB], xb[MSUB], b0[2], b1[2], b2[2];
    Words w = read_words(c, smem, g0, 0, wn);
    read_x(c, smem, g0, 0, row0, xa);
#pragma unroll
    for (int i = 0; i < 4; ++i) pair<0>(w, i, b0);
    for (int g = g0; g < G - 1; ++g) {
      step(xa, w, b0, b1, b2, acc, [&] {
        w = read_words(c, smem, g, 1, wn);
        read_x(c, smem, g, 1, row0, xb);
      });
      step(xb, w, b1, b0, b2, acc, [&] {
        // group g + 1 landed (copies of NS - 2 groups after it may be in flight); all reads of stage g are done
        qmoe_gemm::wait_vmem<(NS - 2) * kCopies>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        Way::barrier();
        copy(c, min(g + NS, G - 1));  // past the end: the last group again, the same bytes to where they are
        w = read_words(c, smem, g + 1, 0, wn);
        read_x(c, smem, g + 1, 0, row0, xa);
      });
    }
    step(xa, w, b0, b1, b2, acc, [&] {
      w = read_words(c, smem, G - 1, 1, wn);
      read_x(c, smem, G - 1, 1, row0, xb);
    });
    step(xb, w, b1, b0, b2, acc, [] {});
    }
    qmoe_gemm::wait_vmem<0>();
    const int lane = fresh_tid() % 64, l16 = lane % 16, q = lane / 16;
    if constexpr (SPLIT) {
      __syncthreads();  // no wave reads its ring any more
      char* ep = block_smem + wave * kRows * 512;
#pragma unroll
      for (int i = 0; i < MSUB; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int v = 0; v < 2; ++v)
            *reinterpret_cast<f32x4_t*>(ep + part_at(16 * i + l16, 2 * (4 * q + t) + v)) =
                f32x4_t{acc[i][4 * v][t], acc[i][4 * v + 1][t], acc[i][4 * v + 2][t], acc[i][4 * v + 3][t]};
      __syncthreads();
      store_parts<kRows>(a, block_smem, u, a.K);
      return;
    }
    if (a.out_f32) {
#pragma unroll
      for (int i = 0; i < MSUB; ++i) {
        const int r = row0 + 16 * i + l16;
        if (r >= u.valid) continue;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int64_t o = u.o0 + 128 * wn + 8 * (4 * q + t);
          if (o >= a.K) continue;
          f32x4_t* out = reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + (u.row0 + r) * a.K + o);
          out[0] = f32x4_t{acc[i][0][t], acc[i][1][t], acc[i][2][t], acc[i][3][t]};
          out[1] = f32x4_t{acc[i][4][t], acc[i][5][t], acc[i][6][t], acc[i][7][t]};
        }
      }
      return;
    }
#pragma unroll
    for (int p = 0; p < (MSUB + 1) / 2; ++p) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int i = 2 * p + v, lr = 32 * wm + 16 * v + l16;
        if (i >= MSUB) break;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int gi = 2 * (16 * wn + 4 * q + t);
          uint4 o;
          o.x = qmoe_gemm::cvt_pk_bf16(acc[i][0][t], acc[i][1][t]);
          o.y = qmoe_gemm::cvt_pk_bf16(acc[i][2][t], acc[i][3][t]);
          o.z = qmoe_gemm::cvt_pk_bf16(acc[i][4][t], acc[i][5][t]);
          o.w = qmoe_gemm::cvt_pk_bf16(acc[i][6][t], acc[i][7][t]);
          *reinterpret_cast<uint4*>(smem + lr * 512 + (gi ^ (2 * (lr % 32))) * 8) = o;
        }
      }
      __syncthreads();
      store_rows<2, 16 * MSUB>(a, smem, u, a.K, p);
    }
  }
};

// ------------------------------------------------------- x W^T, both mxfp4
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes both operands as codes, 16 bytes of
// one block per lane, and a scale byte for each; nothing is converted.
// Contraction in groups of 128.  A lane's scale byte at step kk is block 2kk +
// h of its row: the row's four bytes shifted by h, byte 2kk picked by the
// instruction.
//
// Where the scales are copied from rows, every lane of a copy reads a cache
// line of its own, as many lines for a group's 1.5 KiB of scales as for its 24
// KiB of codes; kLines reads them from lines of consecutive rows (4096^3: 68 ->
// 49 us; 1531 tokens x top-10 of 256 experts: 104 -> 92 us; the lines are made
// with the activations' codes, 12 and 10 us where the codes alone take 9 and 5).
enum { kBytes = 0, kWords = 1, kLines = 2 };
template <int SC, int MSUB, bool SPLIT>
struct QQ {
  static constexpr bool S4 = SC != kBytes;  // a group's four scale bytes of a row at a time
  typedef Geo<SPLIT> Way;
  static constexpr int kCols = Way::kCols, kRows = (SPLIT ? 32 : 64) * MSUB;
  static constexpr int kScaleRows = SPLIT ? 64 : kTileRows;  // rows whose scales are copied: whole waves' worth
  static constexpr int kA = kRows * 64, kB = kCols * 64;
  static constexpr int kSA = kScaleRows * (S4 ? 4 : 16), kSB = kCols * (S4 ? 4 : 16);
  static constexpr int kBOff = kA, kSAOff = kBOff + kB, kSBOff = kSAOff + kSA, kStage = kSBOff + kSB;
  static constexpr int NS = S4 ? 3 : 2;
  static constexpr int kRing = NS * kStage;
  static constexpr int kACopies = kRows / 16 / Way::kWaves, kBCopies = kCols / 16 / Way::kWaves;
  static constexpr int kSCopies = kCols / 64 / Way::kWaves;
  static constexpr int kCopies = kACopies + kBCopies + (1 + kSCopies) * (S4 ? 1 : 4);

  struct Ctx {
    RowSrc<kACopies, 4, Way::kWaves> x;
    const char *w, *s, *xs;
    int64_t sline, xline;  // kLines: bytes from a group's line to the next one's
    uint32_t xoff;
    uint32_t woff[kBCopies], soff[kSCopies];
    int wunit;
    uint32_t lds;
    int wave, lane, units;  // wave: of those that fill the ring
  };

  static __device__ __forceinline__ void copy(const Ctx& c, int g, int stage) {
    const uint32_t st = c.lds + stage * kStage;
    const bool whole = 4 * (g + 1) <= c.units;
#pragma unroll
    for (int d = 0; d < kACopies; ++d) {
      const char* p = c.x.p[d] + (size_t)g * 64;
      if (!whole && 4 * g + c.x.unit(d) >= c.units) p = reinterpret_cast<const char*>(zero_page);
      qmoe_gemm::dma16(p, st + (d * Way::kWaves + c.wave) * 1024);
    }
#pragma unroll
    for (int d = 0; d < kBCopies; ++d) {
      const uint32_t dst = st + kBOff + (d * Way::kWaves + c.wave) * 1024;
      if (whole) {
        qmoe_gemm::dma16s(c.w + (size_t)g * 64, c.woff[d], dst);
      } else {
        const char* q = c.w + (size_t)g * 64 + c.woff[d];
        if (4 * g + c.wunit >= c.units) q = reinterpret_cast<const char*>(zero_page);
        qmoe_gemm::dma16(q, dst);
      }
    }
    const uint32_t sa = st + kSAOff + (c.wave & 1) * 256, sb = st + kSBOff + c.wave * 256;
    if constexpr (SC == kLines) {
      qmoe_gemm::dma4s(c.xs + g * c.xline, c.xoff, sa);
#pragma unroll
      for (int d = 0; d < kSCopies; ++d) qmoe_gemm::dma4s(c.s + g * c.sline, c.soff[d], sb + d * 256);
    } else if constexpr (S4) {
      qmoe_gemm::dma4(c.xs + (size_t)g * 4, sa);
#pragma unroll
      for (int d = 0; d < kSCopies; ++d) qmoe_gemm::dma4s(c.s + (size_t)g * 4, c.soff[d], sb + d * 256);
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const bool in = 4 * g + b < c.units;
        dma1(in ? c.xs + (size_t)g * 4 + b : reinterpret_cast<const char*>(zero_page), sa + b * kScaleRows * 4);
#pragma unroll
        for (int d = 0; d < kSCopies; ++d) {
          if (in) dma1s(c.s + (size_t)g * 4 + b, c.soff[d], sb + b * kCols * 4 + d * 256);
          else dma1(zero_page, sb + b * kCols * 4 + d * 256);
        }
      }
    }
  }

  // A row's four scale bytes in group g, those of lane half h at bytes 0 and 2.
  static __device__ __forceinline__ int scales(const char* st, int rows, int row, int h) {
    if constexpr (S4) {
      return (int)(*reinterpret_cast<const uint32_t*>(st + row * 4) >> (8 * h));
    } else {
      const uint32_t lo = *reinterpret_cast<const uint32_t*>(st + (h * rows + row) * 4);
      const uint32_t hi = *reinterpret_cast<const uint32_t*>(st + ((2 + h) * rows + row) * 4);
      return (int)(lo | (hi << 16));
    }
  }
  static __device__ __forceinline__ void read_scales(const char* st, int row, int col, int h, int (&sa)[MSUB],
                                                     int (&sb)[4]) {
#pragma unroll
    for (int i = 0; i < MSUB; ++i) sa[i] = scales(st + kSAOff, kScaleRows, row + 32 * i, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) sb[j] = scales(st + kSBOff, kCols, col + 32 * j, h);
  }
  struct Frag {
    i32x4_t a[MSUB], b[4];
  };
  static __device__ __forceinline__ void read(const Ctx& c, const char* st, int kk, int row0, int col0, Frag& f) {
    const int l32 = c.lane % 32, unit = (2 * kk + c.lane / 32) ^ swz4(l32);  // swz4 repeats every 16 rows
#pragma unroll
    for (int i = 0; i < MSUB; ++i)
      f.a[i] = *reinterpret_cast<const i32x4_t*>(st + (row0 + 32 * i + l32) * 64 + unit * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f.b[j] = *reinterpret_cast<const i32x4_t*>(st + kBOff + (col0 + 32 * j + l32) * 64 + unit * 16);
  }
  typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;
  static __device__ __forceinline__ i32x8_t wide(const i32x4_t& v) {
    return i32x8_t{v[0], v[1], v[2], v[3], 0, 0, 0, 0};  // the fp4 form reads the first four registers
  }
  template <int KK>
  static __device__ __forceinline__ void products(const Frag& f, const int (&sa)[MSUB], const int (&sb)[4],
                                                  f32x16_t (&acc)[MSUB][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < MSUB; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f.b[j]), wide(f.a[i]), acc[i][j], 4, 4,
                                                                    2 * KK, sb[j], 2 * KK, sa[i]);
  }

  static __device__ __forceinline__ void run(const GemmArgs& a, const Unit& u, char* block_smem) {
    Ctx c;
    const int tid = fresh_tid();
    c.lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = SPLIT ? 0 : wave / 2, wn = SPLIT ? 0 : wave % 2;
    char* smem = block_smem + (SPLIT ? wave * kRing : 0);
    c.wave = SPLIT ? 0 : wave;
    c.units = (int)(a.K / kBlock);
    c.lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)smem);
    c.x = row_sources<kACopies, 4, Way::kWaves>(a, u, a.xq, (int64_t)c.units * 16, c.wave, c.lane);
    {
      const int64_t i = u.row0 + min((c.wave & 1) * 64 + c.lane, u.valid - 1);
      const int64_t x = min(max(a.x_rows ? (int64_t)a.x_rows[i] : i, (int64_t)0), a.n_x - 1);
      if constexpr (SC == kLines) {
        c.xs = reinterpret_cast<const char*>(a.xl);
        c.xoff = (uint32_t)x * 4;
        c.xline = a.n_x * 4;
        c.sline = a.N * 4;
      } else {
        c.xs = reinterpret_cast<const char*>(a.xs) + x * c.units;
      }
    }
    const int64_t row = (int64_t)u.e * a.N + u.o0;
    const int cols = (int)min((int64_t)kCols, a.N - u.o0);
    c.w = reinterpret_cast<const char*>(a.w) + qmoe_gemm::uniform64(row * c.units * 16);
    if constexpr (SC == kLines)
      c.s = reinterpret_cast<const char*>(a.sl) + qmoe_gemm::uniform64(((int64_t)u.e * ((c.units + 3) / 4) * a.N + u.o0) * 4);
    else
      c.s = reinterpret_cast<const char*>(a.s) + qmoe_gemm::uniform64(row * c.units);
    c.wunit = (c.lane % 4) ^ swz4(c.lane / 4);  // swz4 repeats every 16 columns
#pragma unroll
    for (int d = 0; d < kBCopies; ++d) {
      const int col = (d * Way::kWaves + c.wave) * 16 + c.lane / 4;
      c.woff[d] = (uint32_t)(min(col, cols - 1) * c.units * 16 + c.wunit * 16);
    }
#pragma unroll
    for (int d = 0; d < kSCopies; ++d)
      c.soff[d] = (uint32_t)(min((d * Way::kWaves + c.wave) * 64 + c.lane, cols - 1) * (SC == kLines ? 4 : c.units));
    int g0, G;  // this wave's groups
    Way::template part<1>((c.units + 3) / 4, wave, &g0, &G);
    const int row0 = 32 * MSUB * wm, col0 = 128 * wn;
    const int l32 = c.lane % 32, h = c.lane / 32;

    f32x16_t acc[MSUB][4] = {};
    if (!SPLIT || g0 < G) {
      // past the end: the last group again, into stages that nothing reads any more
#pragma unroll
      for (int i = 0; i < NS; ++i) copy(c, min(g0 + i, G - 1), i);
      qmoe_gemm::wait_vmem<(NS - 1) * kCopies>();
      Way::barrier();
      Frag fa, fb;
      int sa[MSUB], sb[4];
      read(c, smem, 0, row0, col0, fa);
      int at = 0;
      for (int g = g0; g < G; ++g) {
        const char* st = smem + at * kStage;
        read_scales(st, row0 + l32, col0 + l32, h, sa, sb);
        read(c, st, 1, row0, col0, fb);
        products<0>(fa, sa, sb, acc);
        __builtin_amdgcn_sched_barrier(0);
        at = at + 1 == NS ? 0 : at + 1;
        if (g + 1 < G) {
          qmoe_gemm::wait_vmem<(NS - 2) * kCopies>();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          Way::barrier();
          copy(c, min(g + NS, G - 1), at == 0 ? NS - 1 : at - 1);
          read(c, smem + at * kStage, 0, row0, col0, fa);
        }
        __builtin_amdgcn_sched_barrier(0);
        products<1>(fb, sa, sb, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    qmoe_gemm::wait_vmem<0>();
    const int el = fresh_tid() % 64, e32 = el % 32, eh = el / 32;
    if constexpr (SPLIT) {
      Fwd<true, 1, MSUB, true>::put_parts(block_smem + wave * kRows * 512, e32, eh, acc);
      __syncthreads();
      store_parts<kRows>(a, block_smem, u, a.N);
      return;
    }
#pragma unroll
    for (int i = 0; i < MSUB; ++i) {
      __syncthreads();
      const int lr = 32 * wm + e32;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const int gi = (col0 + 32 * j + 2 * v + 4 * eh) / 4;
          *reinterpret_cast<uint2*>(smem + lr * 512 + (gi ^ (2 * e32)) * 8) =
              make_uint2(qmoe_gemm::cvt_pk_bf16(acc[i][j][v], acc[i][j][v + 1]),
                         qmoe_gemm::cvt_pk_bf16(acc[i][j][v + 2], acc[i][j][v + 3]));
        }
      __syncthreads();
      store_rows<2, 32 * MSUB>(a, smem, u, a.N, i);
    }
  }
};

// The forms of a unit by its rows, widest first, each for units of more rows than the next takes.
template <class... Forms>
struct Pick;
template <class F>
struct Pick<F> {
  static constexpr int kRing = F::kRing;
  static __device__ __forceinline__ void run(const GemmArgs& a, const Unit& u, char* smem) { F::run(a, u, smem); }
};
template <class F, class G, class... Rest>
struct Pick<F, G, Rest...> {
  typedef Pick<G, Rest...> Next;
  static constexpr int kRing = F::kRing > Next::kRing ? F::kRing : Next::kRing;
  static __device__ __forceinline__ void run(const GemmArgs& a, const Unit& u, char* smem) {
    if (u.valid > G::kRows) F::run(a, u, smem);
    else Next::run(a, u, smem);
  }
};
template <int MODE, int SC, bool SPLIT>
struct Kernel;
template <int SC>
struct Kernel<kFwd, SC, false> {
  typedef Pick<Fwd<SC == kWords, 2, 2, false>, Fwd<SC == kWords, 1, 3, false>, Fwd<SC == kWords, 1, 2, false>, Fwd<SC == kWords, 1, 1, false>> Forms;
};
template <int SC>
struct Kernel<kFwd, SC, true> {
  typedef Pick<Fwd<SC == kWords, 1, 2, true>, Fwd<SC == kWords, 1, 1, true>> Forms;
};
template <int SC>
struct Kernel<kT, SC, false> {
  typedef Pick<Trn<SC == kWords, 4, false>, Trn<SC == kWords, 3, false>, Trn<SC == kWords, 2, false>, Trn<SC == kWords, 1, false>> Forms;
};
template <int SC>
struct Kernel<kT, SC, true> {
  typedef Pick<Trn<SC == kWords, 4, true>, Trn<SC == kWords, 2, true>, Trn<SC == kWords, 1, true>> Forms;
};
template <int SC, bool SPLIT>
struct Kernel<kQQ, SC, SPLIT> {
  typedef Pick<QQ<SC, 2, SPLIT>, QQ<SC, 1, SPLIT>> Forms;
};

template <int MODE, int SC, bool SPLIT>
__global__ __launch_bounds__(256, SPLIT ? 1 : 2) void mx_gemm_kernel(GemmArgs a, int64_t dense_tiles, int NB) {
  typedef typename Kernel<MODE, SC, SPLIT>::Forms Forms;
  typedef Geo<SPLIT> Way;
  constexpr int kEnd = SPLIT ? 4 * 64 * 512 : 64 * 512;  // the epilogue's rows
  constexpr int kRing = Way::kRings * Forms::kRing > kEnd ? Way::kRings * Forms::kRing : kEnd;
  static_assert(kRing >= 4 * qmoe_gemm::kMaxOrder, "the ranking's scratch");
  static_assert((SPLIT ? 1 : 2) * (kRing + 4 * qmoe_gemm::kMaxOrder) <= kLdsCU, "LDS per CU");
  __shared__ __attribute__((aligned(16))) char smem[kRing];
  __shared__ int order[qmoe_gemm::kMaxOrder];
  const int64_t tiles = a.offsets ? (int64_t)max(a.ntiles[0], 0) : dense_tiles;
  const bool ranked = a.offsets && tiles <= qmoe_gemm::kMaxOrder;
  if (ranked) {
    const qmoe_gemm::Tiles table{a.offsets, a.tile_row, a.tile_exp, a.ntiles, a.n_rows, a.num_experts};
    qmoe_gemm::rank_tiles(table, (int)tiles, order, reinterpret_cast<int*>(smem));
  }
  // a split unit is half a tile
  const int per = SPLIT ? 2 * NB : NB;
  const qmoe_gemm::Snake snake(tiles * per);
  for (int64_t k = 0;; ++k) {
    const int64_t at = snake.unit(k);
    if (at < 0) break;
    int64_t tile = at / per;
    const int sub = (int)(at % per);
    if (ranked) tile = order[tile];
    qmoe_gemm::TileRows t = tile_of(a, tile);
    if constexpr (SPLIT) {
      if (sub >= NB) t.row0 += kRowsHalf, t.valid -= kRowsHalf;
      t.valid = min(t.valid, kRowsHalf);
    }
    if (t.valid <= 0) continue;
    Unit u;
    u.e = __builtin_amdgcn_readfirstlane(t.e);
    u.valid = __builtin_amdgcn_readfirstlane(t.valid);
    u.row0 = qmoe_gemm::uniform64(t.row0);
    u.o0 = (int64_t)__builtin_amdgcn_readfirstlane(SPLIT ? sub % NB : sub) * Way::kCols;
    Forms::run(a, u, smem);
    __syncthreads();  // the ring is free for the next unit
  }
}

template <int MODE, bool SPLIT>
void launch_way(const GemmArgs& a, int64_t max_tiles, hipStream_t st) {
  const int64_t O = MODE == kT ? a.K : a.N;
  const int64_t dense = (a.n_rows + kTileRows - 1) / kTileRows;
  const int64_t NB = (O + Geo<SPLIT>::kCols - 1) / Geo<SPLIT>::kCols;
  const int64_t units = (a.offsets ? max_tiles : dense) * NB * (SPLIT ? 2 : 1);
  const dim3 grid((unsigned)qmoe_gemm::grid_blocks(units, SPLIT ? 1 : 2)), block(256);
  if constexpr (MODE == kQQ) {
    if (a.sl) {
      mx_gemm_kernel<MODE, kLines, SPLIT><<<grid, block, 0, st>>>(a, dense, (int)NB);
      return;
    }
  }
  const bool s4 = a.K % 128 == 0 && qmoe::aligned4(a.s) && (MODE != kQQ || qmoe::aligned4(a.xs));
  if (s4) mx_gemm_kernel<MODE, kWords, SPLIT><<<grid, block, 0, st>>>(a, dense, (int)NB);
  else mx_gemm_kernel<MODE, kBytes, SPLIT><<<grid, block, 0, st>>>(a, dense, (int)NB);
}

// Wide units from this many on: below, split ones are faster.  At 64, 128 and
// 256 wide units of 4096 x 2048 weights (us, wide / split): forward 29.9 / 18.4,
// 31.0 / 32.0, 33.6 / 56.4; transposed 69.6 / 26.0, 69.6 / 46.5
// (256 units of 1024 x 2048: 24.2 / 41.7); both mxfp4 17.1 / 15.0, 17.7 / 25.3,
// 18.6 / 43.7 (at 96 units 17.5 / 24.6).
constexpr int64_t kWideUnits = 160, kWideUnitsQQ = 96;

template <int MODE>
int launch(const GemmArgs& a, int64_t max_tiles, hipStream_t st) {
  const int64_t O = MODE == kT ? a.K : a.N;
  const int64_t tiles = a.offsets ? std::min(max_tiles, a.n_rows) : (a.n_rows + kTileRows - 1) / kTileRows;
  if (tiles * ((O + kWideCols - 1) / kWideCols) < (MODE == kQQ ? kWideUnitsQQ : kWideUnits))
    launch_way<MODE, true>(a, max_tiles, st);
  else
    launch_way<MODE, false>(a, max_tiles, st);
  return qmoe::launch_status("mx_gemm_kernel");
}

RowsArgs rows_of(const GemmArgs& a) {
  return {a.x, a.xq, a.xs, a.x_rows, a.n_rows, a.n_x, a.ldx, a.w, a.s, a.N, a.K, a.out, a.out_f32};
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
  if (!a.w || !a.s || !a.out || (mode == kQQ ? !a.xq || (!a.xs && !a.sl) : !a.x)) return qmoe::fail(QMOE_ERR_INVALID, "null pointer");
  const bool any = a.offsets || a.tile_row || a.tile_exp || a.ntiles;
  if (any && !(a.offsets && a.tile_row && a.tile_exp && a.ntiles)) return qmoe::fail(QMOE_ERR_INVALID, "half a tile table");
  if (!any && a.num_experts != 1) return qmoe::fail(QMOE_ERR_INVALID, "several experts need a tile table");
  if (!any && !a.x_rows && a.n_x < a.n_rows) return qmoe::fail(QMOE_ERR_INVALID, "fewer activation rows than rows");
  if (any && max_tiles == 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty tile table");
  // a block of 256 weight rows is addressed by 32-bit byte offsets
  if (a.N > 0x7FFFFFFF || a.K > (1 << 23) || a.n_rows > 0x7FFFFFFF || a.n_x > 0x7FFFFFFF || max_tiles > 0x7FFFFFFF)
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
  GemmArgs a{x, nullptr, nullptr, x_rows, n_rows, n_x, ldx, w, scales, num_experts, N, K, nullptr, nullptr,
             offsets, tile_row, tile_exp, ntiles, out, out_dtype == QMOE_FP32};
  bool run;
  const int rc = check(a, transpose ? kFwd : kT, max_tiles, out_dtype, &run);
  if (rc != QMOE_OK || !run) return rc;
  hipStream_t st = qmoe::as_stream(stream);
  if (transpose && !offsets && n_rows <= kFewRows) return rows_product(rows_of(a), false, st);
  return transpose ? launch<kFwd>(a, max_tiles, st) : launch<kT>(a, max_tiles, st);
}

extern "C" int qmoe_mxfp4_gather_qqmm(const uint32_t* xq, const uint8_t* xs, int64_t n_x, const int32_t* x_rows,
                                      int64_t n_rows, const uint32_t* w, const uint8_t* scales, int32_t num_experts,
                                      int64_t N, int64_t K, const int32_t* offsets, const int32_t* tile_row,
                                      const int32_t* tile_exp, const int32_t* ntiles, int64_t max_tiles,
                                      const uint32_t* lines, void* out, void* stream) {
  GemmArgs a{nullptr, xq, xs, x_rows, n_rows, n_x, 0, w, scales, num_experts, N, K, lines, nullptr,
             offsets, tile_row, tile_exp, ntiles, out, 0};
  bool run;
  const int rc = check(a, kQQ, max_tiles, QMOE_BF16, &run);
  if (rc != QMOE_OK || !run) return rc;
  if (lines) {
    if (!qmoe::aligned4(lines)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "lines must be 4-byte aligned");
    if (n_x > (1 << 29)) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "n_x=%lld: too many rows for lines", (long long)n_x);
    a.xl = lines + (int64_t)num_experts * ((K + 127) / 128) * N;
  } else if (!offsets && n_rows <= kFewRows) {
    return rows_product(rows_of(a), true, qmoe::as_stream(stream));
  }
  return launch<kQQ>(a, max_tiles, qmoe::as_stream(stream));
}
