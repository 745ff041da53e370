// Weight gradient of a linear layer from its input in full, for gfx950:
//     W[h][n] = sum over tokens t of x[t][h] * grad[t][n] (+ add[h][n]).
// Both operands lie deep (tccl_product.h): the tokens are the summed index.  The transposed result is the same product with its
// operands exchanged.  Where tiles are few the tokens are split over workgroups, whose sums weight_sum_kernel adds up.
#pragma once

#include "tccl_product.h"
#include "tccl_weight.h"

namespace tccl {

struct WeightFullArgs {
  ProductArgs p;          // M, N: rows and columns of the result, K: tokens
  const char* add;
  char* out;
  float* partial;         // [split][M][ld_partial], where the tokens are split
  int64_t ld_add, ld_out, ld_partial;
  int tiles_m, tiles_n, band;
  int steps, splits, steps_per_split;
  int xcds, per_xcd;
};

#if defined(__HIPCC__)

template <typename T, typename OutT, int kTile>
__global__ __launch_bounds__(512, 2) void weight_full_kernel(WeightFullArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Product<T, kTile, true, true, false> Tile;
  __shared__ __attribute__((aligned(1024))) char full_lds[Tile::kLds];
  // An XCD takes a run of the (split, tile) pairs: tiles of one split read the same rows of the operands.
  const int tiles = a.tiles_m * a.tiles_n, item = (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds;
  if (item >= tiles * a.splits) return;
  const int split = item / tiles;
  const TileCoord at = tile_coords(item - split * tiles, a.tiles_m, a.tiles_n, a.band);
  const int m0 = at.m * kTile, n0 = at.n * kTile, first = split * a.steps_per_split;
  const int steps = a.steps - first < a.steps_per_split ? a.steps - first : a.steps_per_split;
  Tile t(a.p, full_lds);
  typename Tile::Sums acc;
  Tile::clear(acc);
  if (steps > 0) t.run(acc, m0, n0, first, steps);  // (no tokens: a result of zeros, or of what is added)
  const int g = t.lane >> 4;
#pragma unroll
  for (int i = 0; i < Tile::kRows; ++i)
#pragma unroll
    for (int j = 0; j < Tile::kBlocksN; ++j) {
      const int row = m0 + t.out_row(i), col = n0 + t.wn * 64 + 16 * j + 4 * g;
      if (row < a.p.M && col < a.p.N) {
        if (a.splits > 1) {
          put4<float>(acc[i][j], (char*)(a.partial + (int64_t)split * a.p.M * a.ld_partial), row * a.ld_partial + col, a.p.N - col);
        } else {
          if (a.add) acc[i][j] += get4<OutT>(a.add, row * a.ld_add + col, a.p.N - col);
          put4<OutT>(acc[i][j], a.out, row * a.ld_out + col, a.p.N - col);
        }
      }
    }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
