// Products of 8-bit integers with many rows on the matrix cores
// (int8_product.h).  Rows are those of a tile table (sorted by expert), or of
// one expert without a table.
//
// A unit is a block of up to 256 rows of one expert times 256 outputs, computed
// by a block of eight waves, one block per CU.  Its form by its rows: WM x WN
// waves of MSUB x NSUB subtiles of v_mfma_i32_32x32x32_i8 each.  Both operands
// reach LDS by asynchronous copies, 128 bytes of a row at a time (a whole line;
// with 64, twice the requests for the same bytes), into a ring of stages, and
// are read from there as fragments, those of a step during the step before.  The
// barrier that hands over a stage stands before a group's last step, whose
// operands are in registers by then; the copies into the stage that it frees are
// spread between the matrix instructions that follow, since a run of them would
// hold up the wave that issues them.
//
// Blocks are persistent.  Units of a table take two tiles of an expert where it
// has them and they fill the chip, so that its weights are read once for up to 256
// rows, and go heavy-first; those of one matrix go in bands of columns, so that the blocks of
// an XCD share rows and columns in its L2.  A unit's first copies are issued
// before the results of the one before it are stored.
//
// 256 x 256 by eight waves: a wave's 128 x 64 outputs read 6 KiB of fragments for
// 8 matrix instructions (with four waves of 128 x 128 4 for 8, but one wave per
// SIMD waits alone: 75 us at 4096^3 where eight took 65), and a unit copies half the
// bytes per product that 128 x 128 does (both operands pass L2 -> LDS at up to 33 TB/s
// in 128-byte pieces, 17 in 64-byte ones).
//
// 4096^3 takes 61-66 us by the card (2.1-2.25 POP/s), 8192^3 444-462 (2.4-2.5), where
// a loop of the matrix instructions alone reaches 3.42: 40 and 322 us.  Two things keep
// them there: the board is at or near its power limit (1336-1400 of 1400 W; the clock
// falls from 2.4 GHz to 1.69-1.81, the loop's own is 1.77), and at that clock the
// matrix cores are busy in 59% and 66% of the cycles, the rest going to waits (for
// copies and LDS and at barriers, 36-39% of the waves' cycles) and to what stands
// beside the loop of a unit.  Experts: 4096 tokens x top-10 of 256, 2048 -> 1024,
// take 157-165 us (537 MB of weights and 84 of results: 130 at a copy's rate) with the
// matrix cores busy in 30% of the cycles and the waves waiting in 51%, 512 tokens
// 102-111 (109 for the weights alone at a copy's rate, 87 at a stream read's); few rows
// an expert, in tokens: 7 (61 experts) 27.5 us, 16 (101) 51, 32 (147) 74, 64 (201) 96,
// 128 (226) 103, which is 4.2 to 4.7 TB/s of weights.
// Three stages of 128-column units for experts, more in flight but more units:
// 185 us instead of 164; results stored from the registers, with the ring filled
// meanwhile, 170 instead of 165.
#include <algorithm>

#include "gemm_common.h"
#include "int8_few.h"

namespace {

using namespace qmoe_i8;
using qmoe_gemm::kTileRows;

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kPairRows = 2 * kTileRows;  // rows of a unit, at most
constexpr int kGroup = 128;              // bytes of the contraction per stage
constexpr int kUnits = kGroup / 16;      // and its 16-byte units
constexpr int kSteps = kGroup / 32;
constexpr int kRound = kWaves * (1024 / kGroup);  // rows that one copy of every wave fills
constexpr int kMaxACopies = kPairRows / kRound;
constexpr int kLdsCU = 160 * 1024;
// The results are staged in the ring's second 64 KiB: the first stage of the next unit is filled meanwhile.
constexpr int kStaging = 64 * 1024, kRing = 144 * 1024;
__device__ __attribute__((aligned(16))) uint32_t zero_unit[4];  // what copies past the contraction's end read

// The thread's index through an empty asm, so that what is computed from it is
// computed here and not kept in registers across the unit loop.
__device__ __forceinline__ int fresh_tid() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

// All waves of the block are here, and their accesses to LDS are done; memory operations may be under way.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct Unit {
  int e, valid;      // valid 0: none
  int64_t row0, o0;  // first row; first output
};

// The activation row of a unit's row; past the end: the last again, not stored.
__device__ __forceinline__ int64_t row_of(const Product& a, const Unit& u, int row) {
  const int64_t r = u.row0 + min(row, u.valid - 1);
  return min(max(a.x_rows ? (int64_t)a.x_rows[r] : r, (int64_t)0), a.n_x - 1);
}

// Swizzle of a row's eight 16-byte units in LDS: one unit of sixteen
// consecutive rows is read without bank conflicts.
__device__ __forceinline__ int swz(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Sixteen bytes stored at any element's address.
struct __attribute__((packed)) Loose16 {
  i32x4_t v __attribute__((aligned(2)));
};

// The activation rows of a unit that a lane copies from, and whose scale it copies.
struct Rows {
  int x[kMaxACopies], scale;
};
__device__ __forceinline__ Rows rows_of(const Product& a, const Unit& u) {
  const int tid = fresh_tid(), lane = tid % 64, wave = tid / 64;
  Rows r;
#pragma unroll
  for (int d = 0; d < kMaxACopies; ++d) r.x[d] = (int)row_of(a, u, d * kRound + wave * (kRound / kWaves) + lane / kUnits);
  r.scale = (int)row_of(a, u, min(tid, kPairRows - 1));
  return r;
}

template <int COLS>
struct Ctx {
  const char* x[kMaxACopies];  // the lane's unit of each copy's row
  const char* w;               // the unit's columns
  uint32_t woff[COLS / kRound];
  int unit;  // the lane's unit within a group: the rows of its copies swizzle alike
  uint32_t lds;
  int wave, lane, units;
  // What is alike for all lanes of a wave, in scalar registers.
  __device__ __forceinline__ void settle(const Product& a, const char* smem) {
    const int tid = fresh_tid();
    units = (int)(a.K / 16);
    lane = tid % 64;
    wave = __builtin_amdgcn_readfirstlane(tid / 64);
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)smem);
    w = reinterpret_cast<const char*>(qmoe_gemm::uniform64((int64_t)w));
  }
};

// Copy d of group g into the stage at `st`, of the wave's NA of x and those
// of w.  Units past the contraction's end are zeros of x, and of w the group's
// first unit, whatever it holds.
template <int COLS>
__device__ __forceinline__ void copy_x(const Ctx<COLS>& c, int g, uint32_t st, int d) {
  const bool in = g * kUnits + c.unit < c.units;
  const char* p = c.x[d] + (size_t)g * kGroup;
  qmoe_gemm::dma16(in ? p : reinterpret_cast<const char*>(zero_unit), st + (d * kWaves + c.wave) * 1024);
}
template <int COLS>
__device__ __forceinline__ void copy_w(const Ctx<COLS>& c, int g, uint32_t st, int d) {
  const bool in = g * kUnits + c.unit < c.units;
  qmoe_gemm::dma16s(c.w + (size_t)g * kGroup, c.woff[d] - (in ? 0u : (uint32_t)c.unit * 16),
                    st + (d * kWaves + c.wave) * 1024);
}

// A unit's addresses, and the copies of its scales (into s: rows', then columns') and of its first group.
template <class Forms>
__device__ __forceinline__ Ctx<Forms::kCols> begin(const Product& a, const Unit& u, const Rows& rows, char* smem, float* s) {
  constexpr int COLS = Forms::kCols, kBCopies = COLS / kRound;
  Ctx<COLS> c;
  const int tid = fresh_tid();
  const int64_t n0 = (int64_t)u.e * a.N + u.o0;
  const int cols = (int)min((int64_t)COLS, a.N - u.o0);
  c.w = reinterpret_cast<const char*>(a.w) + n0 * a.K;
  c.settle(a, smem);
  c.unit = (c.lane % kUnits) ^ swz(c.wave * (kRound / kWaves) + c.lane / kUnits);
  static_assert(kRound % 16 == 0, "the copies' rows swizzle alike");
#pragma unroll
  for (int d = 0; d < kMaxACopies; ++d)
    c.x[d] = reinterpret_cast<const char*>(a.x) + (int64_t)rows.x[d] * a.K + c.unit * 16;
#pragma unroll
  for (int d = 0; d < kBCopies; ++d)
    c.woff[d] = (uint32_t)(min(d * kRound + c.wave * (kRound / kWaves) + c.lane / kUnits, cols - 1) * (int)a.K + c.unit * 16);
  const uint32_t ls = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)s);
  if (c.wave < kPairRows / 64) {
    qmoe_gemm::dma4(a.sx + rows.scale, ls + c.wave * 256);
    qmoe_gemm::dma4(a.sw + n0 + min(tid, cols - 1), ls + kPairRows * 4 + c.wave * 256);
  }
  static_assert(COLS <= kPairRows, "the same waves copy both scales");
  const int na = Forms::copies(u.valid);
#pragma unroll
  for (int d = 0; d < kMaxACopies; ++d)
    if (d < na) copy_x(c, 0, c.lds, d);
#pragma unroll
  for (int d = 0; d < kBCopies; ++d) copy_w(c, 0, c.lds + na * kWaves * 1024, d);
  return c;
}

// NX stages of a group's x and w, and NW - NX more of w, which comes from further
// away (192 rows on each of 256 experts, three of w beside two of x: 162 -> 152 us).
template <int WM_, int WN_, int MSUB_, int NSUB_, int NX_, int NW_ = NX_>
struct Form {
  static constexpr int WM = WM_, WN = WN_, MSUB = MSUB_, NSUB = NSUB_, NX = NX_, NW = NW_;
  static constexpr int kRows = 32 * WM * MSUB, kCols = 32 * WN * NSUB;
  static constexpr int kBCopies = kCols / kRound, kACopies = (kRows + kRound - 1) / kRound, kCopies = kACopies + kBCopies;  // per wave and group
  static constexpr int kA = kACopies * kWaves * 1024, kB = kCols * kGroup, kStage = kA + kB;
  static constexpr int kAfter = (NX - 2) * kCopies + (NW - NX) * kBCopies;  // copies under way past the group that is waited for
  static_assert(WM * WN == kWaves, "eight waves");
  static_assert(NX * kStage + (NW - NX) * kB <= kRing && kStage <= kStaging && NW - NX <= 1, "the ring");
  typedef i32x16_t Acc[MSUB][NSUB];
  typedef ::Ctx<kCols> Ctx;

  struct Frag {
    i32x4_t a[MSUB], b[NSUB];
  };
  static __device__ __forceinline__ int x_at(int stage) { return stage * kStage; }
  static __device__ __forceinline__ int w_at(int stage) {
    return NW == NX || stage < NX ? stage * kStage + kA : NX * kStage + (stage - NX) * kB;
  }
  static __device__ __forceinline__ void read(const Ctx& c, const char* sx, const char* sw, int kk, int row0, int col0, Frag& f) {
    const int l32 = c.lane % 32, unit = (2 * kk + c.lane / 32) ^ swz(l32);  // swz repeats every 16 rows
#pragma unroll
    for (int i = 0; i < MSUB; ++i)
      f.a[i] = *reinterpret_cast<const i32x4_t*>(sx + (row0 + 32 * i + l32) * kGroup + unit * 16);
#pragma unroll
    for (int j = 0; j < NSUB; ++j)
      f.b[j] = *reinterpret_cast<const i32x4_t*>(sw + (col0 + 32 * j + l32) * kGroup + unit * 16);
  }
  // A step's products with PIECES calls of more(i) spread between them.
  template <int PIECES, class More>
  static __device__ __forceinline__ void products(const Frag& f, Acc& acc, More more) {
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

  // The sums of a unit whose first group is under way; last() is called before the last group's products, between() once
  // nothing reads the ring any more.
  template <class Last, class Between>
  static __device__ __forceinline__ void run(const Product& a, const Unit& u, Ctx& c, char* smem, const float* s,
                                             Last last, Between between) {
    c.settle(a, smem);
    const int row0 = 32 * MSUB * (c.wave / WN), col0 = 32 * NSUB * (c.wave % WN);
    const int G = (c.units + kUnits - 1) / kUnits;
    Acc acc = {};
    if (NW > 2) meet();  // the staging of the unit before, which other stages overlap, is read
    // past the end: the last group again, into stages that nothing reads any more
#pragma unroll
    for (int i = 1; i < NW - 1; ++i) {
      if (i < NX - 1) {
#pragma unroll
        for (int d = 0; d < kACopies; ++d) copy_x(c, min(i, G - 1), c.lds + x_at(i), d);
      }
#pragma unroll
      for (int d = 0; d < kBCopies; ++d) copy_w(c, min(i, G - 1), c.lds + w_at(i), d);
    }
    qmoe_gemm::wait_vmem<kAfter>();
    meet();
    Frag f[2];
    read(c, smem + x_at(0), smem + w_at(0), 0, row0, col0, f[0]);
    int ax = 0, aw = 0;  // the stages of group g
    for (int g = 0; g < G; ++g) {
      if (g + 1 == G) last();
      const char *sx = smem + x_at(ax), *sw = smem + w_at(aw);
      const int fx = ax == 0 ? NX - 1 : ax - 1, fw = NW == NX ? fx : aw == 0 ? NW - 1 : aw - 1;  // freed
      const int gx = min(g + NX - 1, G - 1), gw = min(g + NW - 1, G - 1);
#pragma unroll
      for (int kk = 0; kk + 1 < kSteps; ++kk) {
        read(c, sx, sw, kk + 1, row0, col0, f[(kk + 1) & 1]);
        if (kk == 0)
          products<kCopies>(f[0], acc, [&](int p) {
            if (p < kACopies) copy_x(c, gx, c.lds + x_at(fx), p);
            else copy_w(c, gw, c.lds + w_at(fw), p - kACopies);
          });
        else products<0>(f[kk & 1], acc, [](int) {});
        __builtin_amdgcn_sched_barrier(0);
      }
      ax = ax + 1 == NX ? 0 : ax + 1;
      aw = NW == NX ? ax : aw + 1 == NW ? 0 : aw + 1;
      if (g + 1 < G) {
        // the next group landed (copies of those after it may be in flight); this one's reads are done
        qmoe_gemm::wait_vmem<kAfter>();
        meet();
        read(c, smem + x_at(ax), smem + w_at(aw), 0, row0, col0, f[kSteps & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
      products<0>(f[(kSteps - 1) & 1], acc, [](int) {});
      __builtin_amdgcn_sched_barrier(0);
    }
    qmoe_gemm::wait_vmem<0>();
    meet();
    between();
    if (a.dtype == QMOE_FP32) store<4>(a, u, smem + kStaging, s, acc);
    else store<2>(a, u, smem + kStaging, s, acc);
  }

  // The results through LDS, a row subtile of every wave at a time, so that rows
  // leave in whole lines.  Passes of 2-byte results take the staging's halves in
  // turn: a half is written again only past the barrier of the pass between.
  template <int SIZE>
  static __device__ __forceinline__ void store(const Product& a, const Unit& u, char* staging, const float* s, Acc& acc) {
    constexpr int kPitch = kCols * SIZE, kPer = 16 / SIZE, kRowUnits = kCols / kPer;
    constexpr int kReads = 32 * WM * kRowUnits / kThreads;  // per thread and pass
    const int tid = fresh_tid(), lane = tid % 64, l32 = lane % 32, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), wm = wave / WN, wn = wave % WN;
    const int lr = 32 * wm + l32;
    const int64_t left = a.N - u.o0;
#pragma unroll
    for (int i = 0; i < MSUB; ++i) {
      char* ep = staging + (SIZE == 2 ? (i & 1) * (kStaging / 2) : 0);
      if (SIZE == 4 && i) meet();
      const float sx = s[32 * MSUB * wm + 32 * i + l32];
      const bool plain = __all(ordinary(sx));
#pragma unroll
      for (int j = 0; j < NSUB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const int gi = (32 * NSUB * wn + 32 * j + 2 * v + 4 * h) / 4;  // four outputs
          const f32x4_t sw = *reinterpret_cast<const f32x4_t*>(s + kPairRows + 4 * gi);
          f32x4_t y;
          if (plain) {
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = (float)acc[i][j][v + k] * sx * sw[k];
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = scaled(acc[i][j][v + k], sx, sw[k]);
          }
          if constexpr (SIZE == 4) {
            *reinterpret_cast<f32x4_t*>(ep + lr * kPitch + (gi ^ (l32 % kRowUnits)) * 16) = y;
          } else {
            uint2 o;
            if (a.dtype == QMOE_BF16) {
              o = make_uint2(qmoe_gemm::cvt_pk_bf16(y[0], y[1]), qmoe_gemm::cvt_pk_bf16(y[2], y[3]));
            } else {
              typedef _Float16 h4 __attribute__((ext_vector_type(4)));
              o = __builtin_bit_cast(uint2, h4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]});
            }
            *reinterpret_cast<uint2*>(ep + lr * kPitch + (gi ^ (2 * (l32 % kRowUnits))) * 8) = o;
          }
        }
      meet();
      uint32_t from[kReads];
      i32x4_t v[kReads];
#pragma unroll
      for (int t = 0; t < kReads; ++t) {
        const int r = (t * kThreads + tid) / kRowUnits, unit = (t * kThreads + tid) % kRowUnits;
        from[t] = (uint32_t)(uintptr_t)ep + r * kPitch + (unit ^ (r % 32 % kRowUnits)) * 16;
      }
      lds_read16(v, from);
#pragma unroll
      for (int t = 0; t < kReads; ++t) {
        const int r = (t * kThreads + tid) / kRowUnits, unit = (t * kThreads + tid) % kRowUnits;
        const int row = 32 * MSUB * (r / 32) + 32 * i + r % 32, n = kPer * unit;
        if (row >= u.valid || n >= left) continue;
        char* to = static_cast<char*>(a.out) + ((u.row0 + row) * a.N + u.o0 + n) * SIZE;
        if (a.N % kPer == 0) {
          __builtin_nontemporal_store(v[t], reinterpret_cast<i32x4_t*>(to));
        } else if (n + kPer <= left) {
          reinterpret_cast<Loose16*>(to)->v = v[t];
        } else {
#pragma unroll
          for (int k = 0; k < kPer - 1; ++k) {
            if (n + k >= left) break;
            if constexpr (SIZE == 4) reinterpret_cast<int*>(to)[k] = v[t][k];
            else reinterpret_cast<uint16_t*>(to)[k] = (uint16_t)((uint32_t)v[t][k / 2] >> (16 * (k % 2)));
          }
        }
      }
    }
  }
  template <int N>
  static __device__ __forceinline__ void lds_read16(i32x4_t (&v)[N], const uint32_t (&a)[N]) {
    if constexpr (N == 2) {
      asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(v[0]), "=&v"(v[1]) : "v"(a[0]), "v"(a[1]) : "memory");
    } else {
      qmoe_gemm::lds_read16_all(v, a);
    }
  }
};

// The forms of a unit by its rows, widest first, each for units of more rows than the next takes.
template <class... Forms>
struct Pick;
template <class F>
struct Pick<F> {
  static constexpr int kCols = F::kCols;
  // Copies of activation rows per wave and group of the form for so many rows.
  static __device__ __forceinline__ int copies(int) { return F::kACopies; }
  template <class... A>
  static __device__ __forceinline__ void run(const Product& a, const Unit& u, A&&... rest) { F::run(a, u, rest...); }
};
template <class F, class G, class... Rest>
struct Pick<F, G, Rest...> {
  static constexpr int kCols = F::kCols;
  static_assert(kCols == G::kCols, "forms of one unit");
  static __device__ __forceinline__ int copies(int valid) {
    return valid > G::kRows ? F::kACopies : Pick<G, Rest...>::copies(valid);
  }
  template <class... A>
  static __device__ __forceinline__ void run(const Product& a, const Unit& u, A&&... rest) {
    if (u.valid > G::kRows) F::run(a, u, rest...);
    else Pick<G, Rest...>::run(a, u, rest...);
  }
};
typedef Pick<Form<2, 4, 4, 2, 2>, Form<2, 4, 3, 2, 2, 3>, Form<2, 4, 2, 2, 3>, Form<1, 8, 3, 1, 3>, Form<1, 8, 2, 1, 3>,
             Form<1, 8, 1, 1, 3>> Wide;
// 64 x 128 and 128 x 128 outputs, for products of few units: five and three
// groups ahead, where it is the copies' way that takes the time.
constexpr int kNarrowRows = 64;
typedef Pick<Form<2, 4, 1, 1, 6>> Narrow;
typedef Pick<Form<2, 4, 2, 1, 4>, Form<2, 4, 1, 1, 6>> Middle;

// The rows of a table's row unit: two tiles of an expert (none for the second of
// them), a tile or half of one.
__device__ __forceinline__ qmoe_gemm::TileRows unit_rows_of(const qmoe_gemm::Tiles& t, int unit, int unit_rows) {
  if (unit_rows == kTileRows) return qmoe_gemm::tile_rows_of(t, unit);
  if (unit_rows < kTileRows) {
    qmoe_gemm::TileRows r = qmoe_gemm::tile_rows_of(t, unit / 2);
    const int first = unit % 2 * unit_rows;
    r.row0 += first;
    r.valid = min(r.valid - first, unit_rows);
    return r;
  }
  qmoe_gemm::TileRows r = qmoe_gemm::tile_rows_of(t, unit);
  const int64_t first = t.offsets[r.e], end = min((int64_t)t.offsets[r.e + 1], t.n_rows);
  r.valid = r.valid <= 0 || ((r.row0 - first) / kTileRows) % 2 ? 0 : (int)min((int64_t)kPairRows, end - r.row0);
  return r;
}

// Ranks a table's row units (<= kMaxRanked) by their 32-row subtiles, largest
// first and stable in their order; returns how many have rows.  cls is scratch of
// kMaxRanked + 1 ints.  Called by the whole block.
constexpr int kMaxRanked = 1024;
__device__ inline int rank_units(const qmoe_gemm::Tiles& t, int row_units, int unit_rows, int* order, int* cls) {
  for (int i = threadIdx.x; i < row_units; i += kThreads) cls[i] = (max(unit_rows_of(t, i, unit_rows).valid, 0) + 31) / 32;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const uint64_t below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
    constexpr int kClasses = kPairRows / 32;
    int start[kClasses + 1] = {};
    for (int i = 0; i < row_units; i += 64) {
      const int m = i + lane < row_units ? cls[i + lane] : 0;
#pragma unroll
      for (int k = 1; k <= kClasses; ++k) start[k] += __popcll(__ballot(m == k));
    }
    int sum = 0;
#pragma unroll
    for (int k = kClasses; k >= 1; --k) {
      const int n = start[k];
      start[k] = sum;
      sum += n;
    }
    if (lane == 0) cls[kMaxRanked] = sum;
    for (int i = 0; i < row_units; i += 64) {
      const int m = i + lane < row_units ? cls[i + lane] : 0;
#pragma unroll
      for (int k = 1; k <= kClasses; ++k) {
        const uint64_t same = __ballot(m == k);
        if (m == k) order[start[k] + __popcll(same & below)] = i + lane;
        start[k] += __popcll(same);
      }
    }
  }
  __syncthreads();
  const int units = cls[kMaxRanked];
  __syncthreads();  // cls is free
  return units;
}

// row_units: of one matrix, or as many as a table has room for.
template <class Forms>
__global__ __launch_bounds__(kThreads) void int8_gemm_kernel(Product a, int64_t row_units, int unit_rows, int NB) {
  constexpr int kCols = Forms::kCols;
  __shared__ __attribute__((aligned(16))) char smem[kRing];
  __shared__ __attribute__((aligned(16))) float scales[2][2 * kPairRows];  // of this unit and the next
  __shared__ int order[kMaxRanked];
  static_assert(kRing + sizeof(scales) + sizeof(order) <= kLdsCU, "LDS per CU");
  static_assert(2 * kStaging <= kRing && kRing >= 4 * (kMaxRanked + 1), "the staged results; the ranking's scratch");
  const qmoe_gemm::Tiles table{a.offsets, a.tile_row, a.tile_exp, a.ntiles, a.n_rows, a.num_experts};
  bool ranked = false;
  if (a.offsets) {
    row_units = min((int64_t)max(a.ntiles[0], 0) * (unit_rows < kTileRows ? 2 : 1), row_units);
    ranked = row_units <= kMaxRanked;
    if (ranked) row_units = rank_units(table, (int)row_units, unit_rows, order, reinterpret_cast<int*>(smem));
  }
  const qmoe_gemm::Snake snake(row_units * NB);
  constexpr int kBand = 8;  // column blocks of a band
  // Every second XCD takes its units lightest first, from four rounds on: long
  // units are bound by the matrix cores, short ones by their weights' way from
  // HBM, and so both kinds are under way at once (five rounds, 4096 tokens x
  // top-10 of 256: 174 -> 167 us; two rounds: 60 -> 62).
  const int64_t rounds = (snake.units + snake.P - 1) / snake.P;
  const bool reversed = a.offsets && rounds >= 4 && snake.q / (snake.P / 8) % 2;
  // A table's units of 64 rounds, a lane each, so that the chain of loads that
  // leads to them is waited for once (512 tokens x top-10 of 256: 104 -> 102 us;
  // 4096 tokens of 512 values 132 -> 125).
  struct Planned {
    int e, valid, row0, col;
  };
  const auto plan = [&](int64_t first) {
    const int64_t r = first + threadIdx.x % 64, at = r < rounds ? snake.unit(reversed ? rounds - 1 - r : r) : -1;
    if (at < 0) return Planned{0, 0, 0, 0};
    const int64_t unit = at / NB;
    const qmoe_gemm::TileRows t = unit_rows_of(table, ranked ? order[unit] : (int)unit, unit_rows);
    return Planned{t.e, t.valid, (int)t.row0, (int)(at % NB)};
  };
  Planned planned{0, 0, 0, 0};
  int64_t round = 0;
  const auto next = [&] {  // this block's next unit
    while (round < rounds) {
      const int64_t r = round++;
      Planned p;
      if (a.offsets) {
        const int lane = (int)(r % 64);
        if (lane == 0) planned = plan(r);
        p = {__builtin_amdgcn_readlane(planned.e, lane), __builtin_amdgcn_readlane(planned.valid, lane),
             __builtin_amdgcn_readlane(planned.row0, lane), __builtin_amdgcn_readlane(planned.col, lane)};
      } else {
        const int64_t at = snake.unit(r);
        if (at < 0) continue;
        const int64_t band = at / (row_units * kBand), in = at % (row_units * kBand);
        const int wide = (int)min((int64_t)kBand, NB - band * kBand);
        const int64_t row0 = in / wide * unit_rows;
        p = {0, (int)min((int64_t)unit_rows, a.n_rows - row0), (int)row0, (int)(band * kBand + in % wide)};
      }
      p.valid = __builtin_amdgcn_readfirstlane(p.valid);
      if (p.valid > 0)
        return Unit{__builtin_amdgcn_readfirstlane(p.e), p.valid, (int64_t)__builtin_amdgcn_readfirstlane(p.row0),
                    (int64_t)__builtin_amdgcn_readfirstlane(p.col) * kCols};
    }
    return Unit{0, 0, 0, 0};
  };
  Unit u = next();
  if (u.valid <= 0) return;
  Ctx<kCols> c = begin<Forms>(a, u, rows_of(a, u), smem, scales[0]);
  for (int s = 0;; s ^= 1) {
    const Unit v = next();
    Rows rows = {};
    Ctx<kCols> d;
    Forms::run(a, u, c, smem, scales[s], [&] { if (v.valid > 0) rows = rows_of(a, v); }, [&] {
      if (v.valid > 0) d = begin<Forms>(a, v, rows, smem, scales[s ^ 1]);
    });
    if (v.valid <= 0) break;
    u = v;
    c = d;
  }
}

template <class Forms>
int launch(const Product& a, int64_t max_tiles, int unit_rows, hipStream_t st) {
  const int64_t NB = (a.N + Forms::kCols - 1) / Forms::kCols, rows = a.offsets ? max_tiles * (unit_rows < kTileRows ? 2 : 1) : (a.n_rows + unit_rows - 1) / unit_rows;
  const dim3 grid((unsigned)qmoe_gemm::grid_blocks(rows * NB, 1));
  int8_gemm_kernel<Forms><<<grid, dim3(kThreads), 0, st>>>(a, rows, unit_rows, (int)NB);
  return qmoe::launch_status("int8_gemm_kernel");
}

// One matrix.  Up to kFewBlocks blocks of 32 x 32 outputs are the few-rows
// kernel's, which splits the contraction (4096 x 2048 weights, 128 / 160 / 192 / 224
// rows: 9.4 / 10.9 / 11.7 / 12.9 us, in 64 x 128 units 11.7 / 11.4 / 11.7 / 11.3;
// 1000 rows of 520 x 1600 9.2 and 10.1, of 520 x 4096 15.8 and 15.7; 3000 rows of
// 215 x 4096 19.6 and 15.7; 100 rows of 2048 x 4096 8.3 and 15.4).  Beyond, the form
// whose rounds of 256 units cost least.  A round's cost, as measured with K = 2048:
// 64 x 128 units 9.5 us, 128 x 128 13, 128 x 256 19, 256 x 256 33; a product of one
// round takes 3 more (N = 4096: 512 rows 12.1 / 13.7 / 18.9 / 29.1 us, 1024 rows 21.0 /
// 15.3 / 18.1 / 29.2, 4096 rows 73 / 55 / 44.5 / 37.6).
constexpr int64_t kFewBlocks = 544, kRoundUnits = 256;
int dense(const Product& a, hipStream_t st) {
  const auto blocks = [&](int64_t rows, int64_t cols) { return (a.n_rows + rows - 1) / rows * ((a.N + cols - 1) / cols); };
  if (blocks(32, 32) <= kFewBlocks) return few_product(a, st);
  const auto cost = [&](int64_t rows, int64_t cols, int64_t round) {
    return (blocks(rows, cols) + kRoundUnits - 1) / kRoundUnits * round;
  };
  const int64_t narrow = cost(kNarrowRows, 128, 19), middle = cost(kTileRows, 128, 26), tall = cost(kTileRows, 256, 38),
                wide = cost(kPairRows, 256, 66), least = std::min({narrow, middle, tall, wide});
  if (least == wide) return launch<Wide>(a, 0, kPairRows, st);
  if (least == tall) return launch<Wide>(a, 0, kTileRows, st);
  return least == middle ? launch<Middle>(a, 0, kTileRows, st) : launch<Narrow>(a, 0, kNarrowRows, st);
}

// A table's rows.  The smallest units that one round of the chip takes, by the
// units that n rows make on as many experts as they can reach, each with half a
// unit to spare; where none are, the widest (64 x 128 / 128 x 128 / 128 x 256 / 256
// x 256, us per call in a graph: 2300 rows on 6 experts, 2016 -> 520 13.2 / 15.8 /
// 20.9 / 34.8; 1860 on 7, 1744 -> 912 19.8 / 16.2 / 21.1 / 34.3; 9500 on 17, 800 ->
// 472 21.5 / 19.8 / 15.5 / 23.7; past a round 8200 on 32, 2048 -> 1024 55 / 45 / 44 /
// 44; 41,000 on 256 - / - / 177 / 164).
int grouped(const Product& a, int64_t max_tiles, hipStream_t st) {
  const int64_t experts = std::min<int64_t>(a.num_experts, a.n_rows);
  const auto fits = [&](int64_t rows, int64_t cols) {
    const int64_t units = std::max(experts, (a.n_rows + rows * experts / 2 + rows - 1) / rows);
    return units * ((a.N + cols - 1) / cols) <= kRoundUnits;
  };
  if (fits(kNarrowRows, 128)) return launch<Narrow>(a, max_tiles, kNarrowRows, st);
  if (fits(kTileRows, 128)) return launch<Middle>(a, max_tiles, kTileRows, st);
  return launch<Wide>(a, max_tiles, fits(kTileRows, 256) ? kTileRows : kPairRows, st);
}

}  // namespace

extern "C" int qmoe_int8_gather_qqmm(const int8_t* x, const float* sx, int64_t n_x, const int32_t* x_rows, int64_t n_rows,
                                     const int8_t* w, const float* sw, int32_t num_experts, int64_t N, int64_t K,
                                     const int32_t* offsets, const int32_t* tile_row, const int32_t* tile_exp,
                                     const int32_t* ntiles, int64_t max_tiles, int out_dtype, void* out, void* stream) {
  Product a{x, sx, x_rows, n_rows, n_x, 1, nullptr, w, sw, num_experts, N, K, offsets, tile_row, tile_exp, ntiles, out, out_dtype};
  bool run;
  const int rc = check(a, false, &run);
  if (rc != QMOE_OK || !run) return rc;
  const bool any = offsets || tile_row || tile_exp || ntiles;
  if (any && !(offsets && tile_row && tile_exp && ntiles)) return qmoe::fail(QMOE_ERR_INVALID, "half a tile table");
  if (!any && num_experts != 1) return qmoe::fail(QMOE_ERR_INVALID, "several experts need a tile table");
  if (!any && !x_rows && n_x < n_rows) return qmoe::fail(QMOE_ERR_INVALID, "fewer activation rows than rows");
  if (any && max_tiles <= 0) return qmoe::fail(QMOE_ERR_INVALID, "an empty tile table");
  if (max_tiles > 0x7FFFFFFF) return qmoe::fail(QMOE_ERR_UNSUPPORTED, "sizes too large");
  hipStream_t st = qmoe::as_stream(stream);
  return any ? grouped(a, max_tiles, st) : dense(a, st);
}
