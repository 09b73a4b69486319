// Order of the tiles and packing of results, shared by the kernels whose persistent CTA pairs walk a list of output tiles.
#pragma once
#include "common.cuh"

namespace cfk {

constexpr int kGemmBand = 8;

__device__ __forceinline__ void tile_coords(int tile, int tiles_r, int tiles_c, int& tr, int& tc, int& batch) {
  const int per_batch = tiles_r * tiles_c;
  batch = tile / per_batch;
  int t = tile - batch * per_batch;
  const int band_tiles = kGemmBand * tiles_c;
  const int band = t / band_tiles;
  const int first_r = band * kGemmBand;
  const int rows_in_band = (tiles_r - first_r) < kGemmBand ? (tiles_r - first_r) : kGemmBand;
  t -= band * band_tiles;
  tr = first_r + t % rows_in_band;
  tc = t / rows_in_band;
  if (band & 1) tc = tiles_c - 1 - tc;   // back and forth: a band starts on the Y panels the band before it ended on
}

__device__ __forceinline__ uint32_t pack_out(bool bf16, float lo, float hi) {
  return bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

}  // namespace cfk
