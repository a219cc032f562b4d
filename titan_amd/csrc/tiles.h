// Tables of tiles by one block of T threads: from the experts' offsets, and from
// their sorted ids.
#pragma once

#include "common.h"

namespace qmoe_tiles {

// Exclusive scan of one value per thread over a block of T threads; also
// returns the total.  Each wave scans its 64 values with shuffles, one wave
// scans the wave totals, and every thread adds its wave's base: three
// barriers.  lds holds at least T / 64 + 1 ints.
template <int T = 1024>
__device__ int block_exclusive_scan(int v, int* lds, int* total) {
  static_assert(T % 64 == 0 && T <= 4096, "whole waves, at most 64");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  constexpr int kWavesPerBlock = T / 64;
  int x = v;  // inclusive scan within the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) lds[w] = x;
  __syncthreads();
  if (w == 0) {
    const int t = lane < kWavesPerBlock ? lds[lane] : 0;
    int u = t;
#pragma unroll
    for (int d = 1; d < kWavesPerBlock; d <<= 1) {
      const int y = __shfl_up(u, d, 64);
      if (lane >= d) u += y;
    }
    if (lane < kWavesPerBlock) lds[lane] = u - t;  // exclusive base of wave `lane`
    if (lane == kWavesPerBlock - 1) lds[kWavesPerBlock] = u;
  }
  __syncthreads();
  *total = lds[kWavesPerBlock];
  const int res = lds[w] + x - v;
  __syncthreads();  // lds is free for the caller's next use
  return res;
}

// Tiles from offsets (offsets[0..E] visible to the block of T threads): one
// (row_start, expert) per tile_rows rows, expert-major; zero-fills
// [ntiles, max_tiles).
template <int T = 1024>
__device__ void emit_tiles(const int32_t* offsets, int E, int tile_rows, int32_t* tile_row,
                           int32_t* tile_exp, int32_t* ntiles, int64_t max_tiles, int* lds) {
  const int tid = threadIdx.x;
  const int seg = (E + T - 1) / T;
  const int lo = min(tid * seg, E), hi = min(lo + seg, E);
  int local = 0;
  for (int e = lo; e < hi; ++e) local += (offsets[e + 1] - offsets[e] + tile_rows - 1) / tile_rows;
  int total;
  int64_t t = block_exclusive_scan<T>(local, lds, &total);
  for (int e = lo; e < hi; ++e) {
    const int s = offsets[e], q = offsets[e + 1];
    for (int r = s; r < q; r += tile_rows, ++t) {
      if (t < max_tiles) {
        tile_row[t] = r;
        tile_exp[t] = e;
      }
    }
  }
  const int64_t nt = min((int64_t)total, max_tiles);
  if (tid == 0) ntiles[0] = (int32_t)nt;
  for (int64_t j = nt + tid; j < max_tiles; j += T) {
    tile_row[j] = 0;
    tile_exp[j] = 0;
  }
}

struct Sorted {
  const int32_t* ids;
  int64_t n;
  int E, tile_rows;
  int32_t *offsets, *tile_row, *tile_exp, *ntiles;
  int64_t max_tiles;
  bool all;  // ids below 0 are expert 0's, ids from E on expert E - 1's, so that every row has a tile
};

constexpr int kSamples = 1024;
// lds: kSamples ints.
template <int T>
__device__ void from_sorted(const Sorted& t, int* lds) {
  static_assert(kSamples % T == 0, "samples by all threads");
  const int64_t n = t.n;
  const int E = t.E;
  // first row whose id >= e, in two levels: a search over every stride-th id,
  // read by the block at once, then one inside a stride.  (Each step of a
  // search in memory is a dependent read, 15 of them at 20,480 rows: 4.8 -> 4.5
  // us per call in a graph, where the ids are in the caches.)
  const int64_t stride = (n + kSamples - 1) / kSamples;
  const int ns = n > 0 ? (int)((n + stride - 1) / stride) : 0;  // samples
#pragma unroll
  for (int i = 0; i < kSamples / T; ++i) {
    const int k = threadIdx.x + i * T;
    if (k < ns) lds[k] = t.ids[k * stride];
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += T) {
    int a = 0, b = ns;
    while (a < b) {
      const int mid = (a + b) >> 1;
      if (lds[mid] < e) a = mid + 1;
      else b = mid;
    }
    // sample a is the first with id >= e: the row lies past sample a - 1
    int64_t lo = a > 0 ? (a - 1) * stride + 1 : 0, hi = min(a * stride, n);
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (t.ids[mid] < e) lo = mid + 1;
      else hi = mid;
    }
    if (t.all && e == 0) lo = 0;
    if (t.all && e == E) lo = n;
    t.offsets[e] = (int32_t)lo;
  }
  __syncthreads();
  emit_tiles<T>(t.offsets, E, t.tile_rows, t.tile_row, t.tile_exp, t.ntiles, t.max_tiles, lds);
}

}  // namespace qmoe_tiles
