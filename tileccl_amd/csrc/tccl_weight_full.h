// Weight gradient of a linear layer from its input in full, for gfx950:
//     W[h][n] = sum over tokens t of x[t][h] * grad[t][n] (+ add[h][n]).
// Both operands lie deep (tccl_product.h): the tokens are the summed index.  The transposed result is the same product with its
// operands exchanged.  Where tiles are few the tokens are split over workgroups, whose sums weight_sum_kernel adds up.
//
// 256 tiles: 8192 x 4096 outputs from 4096 tokens, bf16, 235 us as 16 bits (1.17 PFLOP/s; the vendor library 244 to 248); as fp32 on top of another 252,
// the matrix pipes busy 48 %: 64 + 64 MiB of fp32 behind the last step, which one tile a CU cannot overlap.  128 tiles, like the gated
// layer's, are bound by turns of 0.95 us with one turn's loads under way: 1024 x 512 from 16384 tokens in eight splits 23.5 us, and 4.4 for the sums.
#pragma once

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
  int staged;             // `add` is fp32 with rows on 16 bytes and within reach: add_staged()
  int xcds, per_xcd;
};

#if defined(__HIPCC__)

// A whole 256 x 256 tile of fp32 on top of `add`, whose rows come through LDS in two rounds of 128 (1 KiB each, one load), round 1 while round
// 0 is added and stored: rows of the wavefronts' blocks of either half.  16-byte chunk c of row k lies in slot c ^ (k % 16).
// (Block by block a wavefront would read 64 bytes of 16 rows at a time.)
template <typename Tile>
TCCL_D void add_staged(const WeightFullArgs& a, const Tile& t, typename Tile::Sums& acc, int m0, int n0) {
  const int i16 = t.lane & 15, g = t.lane >> 4;
  const auto from = Tile::window(a.add + ((int64_t)m0 * a.ld_add + n0) * 4, 0xfffffff0ll);
  auto fetch = [&](int r) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      uint32_t off[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int k = 16 * t.wave + 2 * p + o, row = k / 64 * 128 + r * 64 + k % 64;
        off[o] = (uint32_t)(row * a.ld_add * 4) + (uint32_t)((t.lane ^ (k & 15)) * 16);
      }
      char* to = t.lds + (16 * t.wave + 2 * p) * 1024;
      Tile::copy_pair(to, to + 1024, from, off[0], off[1]);
    }
  };
  fetch(0);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    f32x4 more[4][4];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    Tile::barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) more[i][j] = *(const f32x4*)(t.lds + (t.wm * 64 + 16 * i + i16) * 1024 + (((t.wn * 16 + 4 * j + g) ^ i16) * 16));
    if (r == 0) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      Tile::barrier();
      fetch(1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) put4<float>(acc[4 * r + i][j] + more[i][j], a.out, (int64_t)(m0 + t.out_row(4 * r + i)) * a.ld_out + n0 + t.wn * 64 + 16 * j + 4 * g, 4);
  }
}

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
  if constexpr (kTile == 256 && sizeof(OutT) == 4)
    if (a.staged && m0 + kTile <= a.p.M && n0 + kTile <= a.p.N) return add_staged(a, t, acc, m0, n0);
#pragma unroll
  for (int i = 0; i < Tile::kRows; ++i)
#pragma unroll
    for (int j = 0; j < Tile::kBlocksN; ++j) {
      const int64_t row = m0 + t.out_row(i);
      const int col = n0 + t.wn * 64 + 16 * j + 4 * g;
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
