// The gated linear layer, for gfx950:   z = x W = [g | u],   h = act(g) * u,   and from the gradient dh of h
//     dg = dh * u * act'(g),   du = dh * act(g).
//
// Both projections are one product whose B is paired (tccl_product.h): a lane has g and u of the same places in its accumulators, so h,
// and in the backward pass that computes z again dg and du, are made in the epilogue and z is never in memory.  Activations and
// their derivatives are taken in fp32 from the fp32 sums (backward, z kept: from the 16 bits that were kept); what is
// stored is rounded once.
#pragma once

#include "tccl_product.h"

namespace tccl {

enum Activation { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3 };

struct GatedArgs {
  ProductArgs p;        // N: outputs
  char *out, *kept;     // forward: h; z or NULL
  const char* grad;     // backward: dh
  char* inner;          // backward: [dg | du]
  int64_t ld_out, ld_kept, ld_grad, ld_inner;
  int activation;
  int tiles_m, tiles_n, band;
  int xcds, per_xcd;    // dies with an L2 of their own; tiles of one
};

struct GatedGradArgs {
  const char *grad, *kept;
  char* inner;
  int64_t ld_grad, ld_kept, ld_inner;
  int rows, cols, activation;
};

#if defined(__HIPCC__)

TCCL_D float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
TCCL_D float logistic(float x) { return __builtin_amdgcn_rcpf(1.f + exp_of(-x)); }

// act(g) and, if wanted, act'(g).
//
// gelu is g Phi(g).  Phi(-a) = erfcx(a / sqrt 2) exp(-a^2 / 2) / 2 keeps its relative accuracy where Phi is small: erfcx(y) is
// t Q(t) with t = 1 / (1 + y / 2), Q of degree 8 fitted to it over y in [0, 12] (largest relative error 4.4e-8, 4e-7 as it is computed).
// gelu_tanh is g s(2 c (g + k g^3)), s the logistic function: (1 + tanh z) / 2 = s(2 z).  Beyond |g| = 64 s is 0 or 1 and its derivative 0;
// the bound keeps g^3 finite.
template <bool kSlope>
TCCL_D float activated(float g, int activation, float& slope) {
  if (activation == kSilu) {
    const float s = logistic(g);
    if (kSlope) slope = s * (1.f + g * (1.f - s));
    return g * s;
  }
  if (activation == kRelu) {
    if (kSlope) slope = g > 0.f ? 1.f : 0.f;
    return g > 0.f ? g : g == g ? 0.f : g;
  }
  if (activation == kGelu) {
    const float a = fabsf(g), e = exp_of(-0.5f * a * a), t = __builtin_amdgcn_rcpf(1.f + 0.353553390593273762f * a);
    constexpr float q[] = {0.282084465f, 0.282409579f, 0.242853642f, 0.203678414f, -0.028971795f, 0.281474948f, -0.4901793f, 0.286013812f, -0.0593638085f};
    float s = q[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) s = s * t + q[i];
    const float tail = 0.5f * e * t * s, phi = g < 0.f ? tail : 1.f - tail;
    if (kSlope) slope = phi + g * e * 0.398942280401432678f;
    return g * phi;
  }
  constexpr float c = 1.59576912160573071f, k = 0.044715f;  // 2 sqrt(2 / pi)
  const float b = fminf(fmaxf(g, -64.f), 64.f), s = logistic(c * b * (1.f + k * b * b));
  if (kSlope) slope = s + b * s * (1.f - s) * c * (1.f + 3.f * k * b * b);
  return g * s;
}

// Eight neighbouring elements of a row that may start anywhere; `left` (1 ..) of them exist.
template <typename T>
struct Eight {
  typedef T Vec __attribute__((ext_vector_type(8)));
  typedef T Anywhere __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  typedef const Anywhere __attribute__((address_space(1))) From;
  typedef Anywhere __attribute__((address_space(1))) To;
  static TCCL_D Vec get(const char* base, int64_t at, int left) {
    Vec v = {};
    if (left >= 8) {
      v = *(From*)((const T*)base + at);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) v[e] = ((const T*)base)[at + e];
    }
    return v;
  }
  static TCCL_D void put(char* base, int64_t at, int left, Vec v) {
    if (left >= 8) {
      *(To*)((T*)base + at) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) ((T*)base)[at + e] = v[e];
    }
  }
};

// Results leave through LDS, whose rows are then stored whole: out of the accumulators a lane would store 8 bytes of 16 rows each.
// Chunk c (8 elements) of row r of a kWidth wide matrix lies in slot c ^ (r % 16), or r % 8 where a row has 8 chunks: 16 rows that are
// written at a time fall on different banks.
template <typename T, int kTile, bool kBDeep, bool kBackward>
struct Gated : Product<T, kTile, false, kBDeep, true> {
  typedef Product<T, kTile, false, kBDeep, true> Base;
  typedef T Quad __attribute__((ext_vector_type(4)));
  static constexpr int kWidth = kTile / 2, kThreads = Base::kWaves * 64;
  static constexpr int kChunks = kWidth / 8, kMatrix = kTile * kWidth * 2;  // chunks of a row, bytes of a matrix
  const GatedArgs& g;
  TCCL_D Gated(const GatedArgs& args, char* mem) : Base(args.p, mem), g(args) {}

  static TCCL_D char* place(char* matrix, int row, int chunk) { return matrix + row * (kWidth * 2) + ((chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15))) << 4); }
  // This lane's four columns of block column j (0, 1) of block row i.
  TCCL_D char* mine(char* matrix, int i, int j) const {
    const int row = this->wm * (kTile / 2) + 16 * i + (this->lane & 15), col = this->wn * 32 + 16 * j + 4 * (this->lane >> 4);
    return place(matrix, row, col >> 3) + (col & 4) * 2;
  }
  static TCCL_D Quad rounded(f32x4 v) { return (Quad){(T)v[0], (T)v[1], (T)v[2], (T)v[3]}; }

  // A tile's matrix between LDS and rows m0 .. of `base`, columns n0 .. < cols.
  TCCL_D void leave(char* matrix, char* base, int64_t ld, int m0, int64_t n0, int cols) const {
    for (int u = (int)threadIdx.x; u < kTile * kChunks; u += kThreads) {
      const int row = u / kChunks, chunk = u % kChunks;
      if (m0 + row < this->p.M && chunk * 8 < cols)
        Eight<T>::put(base, (int64_t)(m0 + row) * ld + n0 + chunk * 8, cols - chunk * 8, *(const typename Eight<T>::Vec*)place(matrix, row, chunk));
    }
  }
  TCCL_D void enter(char* matrix, const char* base, int64_t ld, int m0, int64_t n0, int cols) const {
    for (int u = (int)threadIdx.x; u < kTile * kChunks; u += kThreads) {
      const int row = u / kChunks, chunk = u % kChunks;
      typename Eight<T>::Vec v = {};
      if (m0 + row < this->p.M && chunk * 8 < cols) v = Eight<T>::get(base, (int64_t)(m0 + row) * ld + n0 + chunk * 8, cols - chunk * 8);
      *(typename Eight<T>::Vec*)place(matrix, row, chunk) = v;
    }
  }

  TCCL_D void tile(int m0, int n0) {
    typename Base::Sums acc;
    Base::clear(acc);
    Base::run(acc, m0, n0, 0, (this->p.K + Base::kStepK - 1) / Base::kStepK);
    char *first = this->lds, *second = this->lds + kMatrix;
    const int cols = this->p.N - n0;
    if constexpr (kBackward) {
      enter(first, g.grad, g.ld_grad, m0, n0, cols);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < Base::kBlocksM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Quad dh = *(const Quad*)mine(first, i, j);
          f32x4 dg, du;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float slope;
            const float a = activated<true>(acc[i][j][e], g.activation, slope), d = (float)dh[e];
            dg[e] = d * acc[i][j + 2][e] * slope;
            du[e] = d * a;
          }
          *(Quad*)mine(first, i, j) = rounded(dg);  // in dh's place: nobody else reads it
          *(Quad*)mine(second, i, j) = rounded(du);
        }
      __syncthreads();
      leave(first, g.inner, g.ld_inner, m0, n0, cols);
      leave(second, g.inner, g.ld_inner, m0, (int64_t)n0 + this->p.N, cols);
    } else {
      if (g.kept) {
#pragma unroll
        for (int i = 0; i < Base::kBlocksM; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            *(Quad*)mine(first, i, j) = rounded(acc[i][j]);
            *(Quad*)mine(second, i, j) = rounded(acc[i][j + 2]);
          }
        __syncthreads();
        leave(first, g.kept, g.ld_kept, m0, n0, cols);
        leave(second, g.kept, g.ld_kept, m0, (int64_t)n0 + this->p.N, cols);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < Base::kBlocksM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f32x4 h;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float none;
            h[e] = activated<false>(acc[i][j][e], g.activation, none) * acc[i][j + 2][e];
          }
          *(Quad*)mine(first, i, j) = rounded(h);
        }
      __syncthreads();
      leave(first, g.out, g.ld_out, m0, n0, cols);
    }
  }
};

template <typename T, int kTile, bool kBDeep, bool kBackward>
__global__ __launch_bounds__(2 * kTile, 2) void gated_kernel(GatedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Gated<T, kTile, kBDeep, kBackward> Tile;
  __shared__ __attribute__((aligned(1024))) char gated_lds[Tile::kLds];
  // Workgroups go to the XCDs in turn; each XCD takes a run of neighbouring tiles, which share their operands in its L2.
  const int id = (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds;
  if (id >= a.tiles_m * a.tiles_n) return;
  const TileCoord at = tile_coords(id, a.tiles_m, a.tiles_n, a.band);
  Tile(a, gated_lds).tile(at.m * kTile, at.n * (kTile / 2));
#endif
}

// dg and du from z as it was kept.  Every value is read once; inner may be kept itself.
template <typename T>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int chunks = (a.cols + 7) / 8;
  const int64_t all = (int64_t)a.rows * chunks;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
    const int64_t row = at / chunks;
    const int col = (int)(at - row * chunks) * 8, left = a.cols - col;
    const typename Eight<T>::Vec dh = Eight<T>::get(a.grad, row * a.ld_grad + col, left), g = Eight<T>::get(a.kept, row * a.ld_kept + col, left),
                                 u = Eight<T>::get(a.kept, row * a.ld_kept + a.cols + col, left);
    typename Eight<T>::Vec dg, du;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope;
      const float act = activated<true>((float)g[e], a.activation, slope), d = (float)dh[e];
      dg[e] = (T)(d * (float)u[e] * slope);
      du[e] = (T)(d * act);
    }
    Eight<T>::put(a.inner, row * a.ld_inner + col, left, dg);
    Eight<T>::put(a.inner, row * a.ld_inner + a.cols + col, left, du);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
