// The gated linear layer, for gfx950:   z = x W = [g | u],   h = act(g) * u,   and from the gradient dh of h
//     dg = dh * u * act'(g),   du = dh * act(g).
//
// Both projections are one product whose B is paired (tccl_product.h): a lane has g and u of the same places in its accumulators, so h,
// and in the backward pass that computes z again dg and du, are made in the epilogue and z is never in memory.  Activations and
// their derivatives are taken in fp32 from the fp32 sums (backward, z kept: from the 16 bits that were kept); what is
// stored is rounded once.
#pragma once

#include "tccl_product.h"
#include "tccl_weight.h"

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
  int first, items;     // tiles ahead of this launch, tiles (of every split) up to its end
  // K split over workgroups: blocks of 64 k in each split, and where their sums go: [split][row][2 N] (NULL: nowhere, a workgroup has them all).
  int splits, blocks_per_split;
  float* partial;
};

struct InputGradArgs {
  ProductArgs p;      // M: tokens, N: inputs, K: both projections
  char* out;
  float* partial;     // [split][M][ld_partial], where K is split
  int64_t ld_out, ld_partial;
  int tiles_m, tiles_n, band;
  int splits, blocks_per_split;
  int xcds, per_xcd, first, items;
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
// t Q(t) with t = 1 / (1 + y / 2), Q of degree 8 fitted to it over y in [0, 12] (largest relative error 6.9e-8 with these coefficients, 4e-7 as it is
// computed; further out exp(-a^2 / 2) is 0).
// gelu_tanh is g s(2 c (g + k g^3)), s the logistic function: (1 + tanh z) / 2 = s(2 z).  Beyond |g| = 64 s is 0 or 1 and its derivative 0;
// the bound keeps g^3 finite (and a NaN what it is).
template <int kAct, bool kSlope>
TCCL_D float activated(float g, float& slope) {
  if (kAct == kSilu) {
    const float s = logistic(g);
    if (kSlope) slope = s * (1.f + g * (1.f - s));
    return g * s;
  }
  if (kAct == kRelu) {
    if (kSlope) slope = g > 0.f ? 1.f : 0.f;
    return g > 0.f ? g : g == g ? 0.f : g;
  }
  if (kAct == kGelu) {
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
  const float b = g < -64.f ? -64.f : g > 64.f ? 64.f : g, s = logistic(c * b * (1.f + k * b * b));
  if (kSlope) slope = s + b * s * (1.f - s) * c * (1.f + 3.f * k * b * b);
  return g * s;
}

template <int kAct>
TCCL_D float activated(float g) {
  float none;
  return activated<kAct, false>(g, none);
}
// One choice for all elements that `body` takes, not one for each.
template <typename Body>
TCCL_D void with_activation(int activation, Body body) {
  switch (activation) {
    case kSilu: return body(std::integral_constant<int, kSilu>{});
    case kGelu: return body(std::integral_constant<int, kGelu>{});
    case kGeluTanh: return body(std::integral_constant<int, kGeluTanh>{});
    default: return body(std::integral_constant<int, kRelu>{});
  }
}

// Results leave through LDS, whose rows are then stored whole: out of the accumulators a lane would store 8 bytes of 16 rows each.
// Chunk c (8 elements) of row r of a kWidth wide matrix lies in slot c ^ (r % 16), or r % 8 where a row has 8 chunks: 16 rows that are
// written at a time fall on different banks.
template <typename T, int kTile, bool kBDeep, bool kBackward>
struct Gated : Product<T, kTile, false, kBDeep, true> {
  typedef Product<T, kTile, false, kBDeep, true> Base;
  typedef T Quad __attribute__((ext_vector_type(4)));
  static constexpr int kWidth = kTile / 2, kThreads = 512;
  static constexpr int kChunks = kWidth / 8, kMatrix = kTile * kWidth * 2;  // chunks of a row, bytes of a matrix
  const GatedArgs& g;
  TCCL_D Gated(const GatedArgs& args, char* mem) : Base(args.p, mem), g(args) {}

  static TCCL_D char* place(char* matrix, int row, int chunk) { return matrix + row * (kWidth * 2) + ((chunk ^ (row & (kChunks < 16 ? kChunks - 1 : 15))) << 4); }
  // This lane's four columns of block column j (0, 1) of block row i.
  TCCL_D char* mine(char* matrix, int i, int j) const {
    const int row = this->out_row(i), col = this->wn * 32 + 16 * j + 4 * (this->lane >> 4);
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

  // A split's sums, for gated_join_kernel.
  TCCL_D void hand_on(const typename Base::Sums& acc, int m0, int n0, int split) const {
    const int64_t n = this->p.N;
#pragma unroll
    for (int i = 0; i < Base::kRows; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t row = m0 + this->out_row(i);
        const int col = n0 + this->wn * 32 + 16 * (j & 1) + 4 * (this->lane >> 4);
        if (row < this->p.M && col < n) put4<float>(acc[i][j], (char*)g.partial, (split * (int64_t)this->p.M + row) * (2 * n) + (j < 2 ? 0 : n) + col, (int)n - col);
      }
  }

  TCCL_D void tile(int m0, int n0, int split) {
    typename Base::Sums acc;
    Base::clear(acc);
    const int begin = split * g.blocks_per_split, all = (this->p.K + Base::kStepK - 1) / Base::kStepK;
    const int steps = all - begin < g.blocks_per_split ? all - begin : g.blocks_per_split;
    if (steps > 0) Base::run(acc, m0, n0, begin, steps);
    if constexpr (kTile == 128)
      if (g.partial) return hand_on(acc, m0, n0, split);
    char *first = this->lds, *second = this->lds + kMatrix;
    const int cols = this->p.N - n0;
    if constexpr (kBackward) {
      enter(first, g.grad, g.ld_grad, m0, n0, cols);
      __syncthreads();
      with_activation(g.activation, [&](auto act) {
#pragma unroll
        for (int i = 0; i < Base::kRows; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Quad dh = *(const Quad*)mine(first, i, j);
            f32x4 dg, du;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float slope;
              const float a = activated<decltype(act)::value, true>(acc[i][j][e], slope), d = (float)dh[e];
              dg[e] = d * acc[i][j + 2][e] * slope;
              du[e] = d * a;
            }
            *(Quad*)mine(first, i, j) = rounded(dg);  // in dh's place: nobody else reads it
            *(Quad*)mine(second, i, j) = rounded(du);
          }
      });
      __syncthreads();
      leave(first, g.inner, g.ld_inner, m0, n0, cols);
      leave(second, g.inner, g.ld_inner, m0, (int64_t)n0 + this->p.N, cols);
    } else {
      if (g.kept) {
#pragma unroll
        for (int i = 0; i < Base::kRows; ++i)
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
      with_activation(g.activation, [&](auto act) {
#pragma unroll
        for (int i = 0; i < Base::kRows; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            f32x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = activated<decltype(act)::value>(acc[i][j][e]) * acc[i][j + 2][e];
            *(Quad*)mine(first, i, j) = rounded(h);
          }
      });
      __syncthreads();
      leave(first, g.out, g.ld_out, m0, n0, cols);
    }
  }
};

// 8192 x 4096 x 8192 bf16, k-major: 803 us, 1.37 PFLOP/s, the matrix pipes busy 67 % of a clock that the load holds at 1.9 GHz (the vendor
// library's product alone 794).  4096 x 4096 x 4096 by rows with z kept 214 us, 1.28 PFLOP/s.  128 tiles take 0.95 us for a turn of 4.2 MFLOP and the 64 KiB
// that it reads, with no other turn's loads under way beneath it and one workgroup a CU: 1003 x 1001 x 1035 16 us.  Of a short sum the start, the
// few steps and the epilogue follow one another with nothing beneath them: 12628 x 208 x 808, gelu, 33 us, backward 47, where memory takes 10 and the vector
// instructions of the activation (silu 13 a value, gelu 25, 30 with its derivative) 8, 13 with the second round that does not fill the device.
template <typename T, int kTile, bool kBDeep, bool kBackward>
__global__ __launch_bounds__(512, 2) void gated_kernel(GatedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Gated<T, kTile, kBDeep, kBackward> Tile;
  __shared__ __attribute__((aligned(1024))) char gated_lds[Tile::kLds];
  // Workgroups go to the XCDs in turn; each XCD takes a run of neighbouring tiles, which share their operands in its L2.
  const int id = a.first + (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds, tiles = a.tiles_m * a.tiles_n;
  if (id >= a.items) return;
  const int split = id / tiles;
  const TileCoord at = tile_coords(id - split * tiles, a.tiles_m, a.tiles_n, a.band);
  Tile(a, gated_lds).tile(at.m * kTile, at.n * (kTile / 2), split);
#endif
}

// Few rows.  The weight is read once and nothing hides its latency but other loads, so a workgroup produces 16 kMB rows x
// 8 kNB outputs (kNB / 2 blocks of 16 columns of either matrix) and its wavefronts share K: each takes every kWaves-th block of 64, requests
// several ahead, turns one from load order to operand order through LDS of its own and adds it up by itself; there is no
// barrier until the sums meet at the end.
//
// Loads have neighbouring lanes on neighbouring addresses.  x and a k-major weight: rows of 128 bytes, chunk c of row r in slot
// c ^ ((r >> 1) & 7).  A weight by rows: of each k row 16 kNB bytes of either matrix, next to each other in LDS; its 32-byte units are permuted
// (unit()) so that the rows that a transposing read touches at a time lie in different banks.
//
// Bound by memory: 1 x 4096 x 8192 bf16, k-major, 24.0 us, 5.6 TB/s, over weights of 2 GiB in turn (over one, which the last-level cache
// holds, 21.2); 13 x 4096 x 4096 fp16 by rows 14.8 us, 4.5 TB/s (rows that are a power of two
// apart lie in few of the L2's channels at a time), and 3 to 4 for the join; in tiles of 32 outputs, that is 64 bytes of a row, 26.
template <typename T, int kMB, int kNB, int kWaves, bool kBDeep>
struct GatedRows {
  typedef typename Mfma<T>::Vec Vec;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 LdsQuad;
  static constexpr int kBudget = (kMB + kNB == 9 ? 160 : 128) / ((kMB + kNB) * 8), kDepth = kBudget > 4 ? 4 : kBudget;  // blocks under way, within the registers there are
  static constexpr int kWaveBytes = (kMB + kNB) * 2048, kSums = kMB * kNB * 256;              // sums of a wavefront
  static constexpr int kLds = kWaves * kWaveBytes > (kWaves + 1) * kSums * 4 ? kWaves * kWaveBytes : (kWaves + 1) * kSums * 4;
  static constexpr int kRowBytes = 32 * kNB, kRowLanes = kRowBytes / 16, kRowsPerLoad = 64 / kRowLanes;  // a k row of a weight by rows
  static constexpr uint32_t kLongest = 0xfffffff0u, kOutside = kLongest;  // bytes of a window; an offset past the end of every one
  struct Block {
    u32x4 x[2 * kMB], w[2 * kNB];
  };

  const GatedArgs& g;
  char* lds;
  const int lane, wave;
  __amdgpu_buffer_rsrc_t rx, rw, ru;
  uint32_t off_x, off_w, pitch_x, pitch_w;

  TCCL_D GatedRows(const GatedArgs& args, char* mem) : g(args), lds(mem), lane((int)(threadIdx.x & 63)), wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))) {}
  static TCCL_D __amdgpu_buffer_rsrc_t window(const char* at, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bytes > (int64_t)kLongest ? kLongest : (uint32_t)bytes, 0x00020000);
  }

  TCCL_D void load(Block& v, int kb) const {
    const int k = g.p.K - kb * 64;  // what is left from this block on
    const bool past = 8 * (lane & 7) >= k;
#pragma unroll
    for (int h = 0; h < 2 * kMB; ++h) v.x[h] = __builtin_amdgcn_raw_buffer_load_b128(rx, past ? kOutside : off_x + (uint32_t)(8 * h) * pitch_x + (uint32_t)kb * 128u, 0, 0);
    if constexpr (kBDeep) {
#pragma unroll
      for (int h = 0; h < 2 * kNB; ++h) {
        const bool none = off_w == kOutside || h * kRowsPerLoad + lane / kRowLanes >= k;
        v.w[h] = __builtin_amdgcn_raw_buffer_load_b128(rw, none ? kOutside : off_w + (uint32_t)(kb * 64 + h * kRowsPerLoad) * pitch_w, 0, kNB == 8 ? kStreaming : 0);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2 * kNB; ++h) {
        const uint32_t o = off_w + (uint32_t)(8 * (h % kNB)) * pitch_w + (uint32_t)kb * 128u;
        v.w[h] = __builtin_amdgcn_raw_buffer_load_b128(h < kNB ? rw : ru, past ? kOutside : o, 0, kStreaming);
      }
    }
  }
  static TCCL_D int unit(int u, int k) { return u ^ (kNB == 8 ? 2 * (k & 3) : kNB == 4 ? k & 2 : 0) ^ ((k >> 3) & 1); }
  // A wavefront's LDS operations execute in the order issued; the fences keep the compiler to it.
  TCCL_D void stage(const Block& v) const {
    asm volatile("" ::: "memory");
    char* at = lds + wave * kWaveBytes;
#pragma unroll
    for (int h = 0; h < 2 * kMB; ++h) {
      const int r = 8 * h + (lane >> 3);
      *(u32x4*)(at + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4)) = v.x[h];
    }
    at += kMB * 2048;
#pragma unroll
    for (int h = 0; h < 2 * kNB; ++h) {
      if constexpr (kBDeep) {
        const int k = h * kRowsPerLoad + lane / kRowLanes, c = lane % kRowLanes;
        *(u32x4*)(at + k * kRowBytes + (unit(c >> 1, k) << 5) + ((c & 1) << 4)) = v.w[h];
      } else {
        const int r = 8 * h + (lane >> 3);
        *(u32x4*)(at + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4)) = v.w[h];
      }
    }
    asm volatile("" ::: "memory");
  }
  TCCL_D Vec by_row(int block, int kh) const {
    const int i = lane & 15;
    return *(const Vec*)(lds + wave * kWaveBytes + block * 2048 + i * 128 + (((4 * kh + (lane >> 4)) ^ ((i >> 1) & 7)) << 4));
  }
  TCCL_D Vec turned(int j, int kh) const {
    const int i = lane & 15, t = i >> 2, cq = i & 3;
    s16x4 half[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = 32 * kh + 8 * (lane >> 4) + 4 * q + t;
      const char* p = lds + wave * kWaveBytes + kMB * 2048 + k * kRowBytes + (unit(j, k) << 5) + cq * 8;
      half[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)p);
    }
    return __builtin_bit_cast(Vec, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  TCCL_D void multiply(f32x4 (&acc)[kMB][kNB]) const {
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      Vec x[kMB], w[kNB];
#pragma unroll
      for (int j = 0; j < kNB; ++j) w[j] = kBDeep ? turned(j, kh) : by_row(kMB + j, kh);
#pragma unroll
      for (int i = 0; i < kMB; ++i) x[i] = by_row(i, kh);
#pragma unroll
      for (int i = 0; i < kMB; ++i)
#pragma unroll
        for (int j = 0; j < kNB; ++j) acc[i][j] = Mfma<T>::run16(w[j], x[i], acc[i][j]);
    }
  }

  TCCL_D void tile(int m0, int n0, int split) {
    const ProductArgs& p = g.p;
    const int left = p.N - n0;
    pitch_x = (uint32_t)(p.lda * 2), pitch_w = (uint32_t)(p.ldb * 2);
    rx = window(p.a + (int64_t)m0 * p.lda * 2, ((int64_t)(p.M - m0 - 1) * p.lda + (p.K + 7) / 8 * 8) * 2);
    off_x = (uint32_t)(lane >> 3) * pitch_x + (uint32_t)(lane & 7) * 16u;
    if constexpr (kBDeep) {
      rw = window(p.b + (int64_t)n0 * 2, ((int64_t)(p.K - 1) * p.ldb + (left + 7) / 8 * 8) * 2 + p.up);
      const int c = lane % kRowLanes;
      off_w = 8 * (c % kNB) < left ? (uint32_t)(lane / kRowLanes) * pitch_w + (uint32_t)((c % kNB) * 16 + (c < kNB ? 0 : p.up)) : kOutside;
    } else {
      const int64_t bytes = ((int64_t)(left - 1) * p.ldb + (p.K + 7) / 8 * 8) * 2;
      rw = window(p.b + (int64_t)n0 * p.ldb * 2, bytes);
      ru = window(p.b + (int64_t)n0 * p.ldb * 2 + p.up, bytes);
      off_w = (uint32_t)(lane >> 3) * pitch_w + (uint32_t)(lane & 7) * 16u;
    }
    f32x4 acc[kMB][kNB];
#pragma unroll
    for (int i = 0; i < kMB; ++i)
#pragma unroll
      for (int j = 0; j < kNB; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int first = split * g.blocks_per_split, all = (p.K + 63) / 64, blocks = first + g.blocks_per_split < all ? first + g.blocks_per_split : all;
    Block v[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (first + wave + d * kWaves < blocks) load(v[d], first + wave + d * kWaves);
    for (int kb = first + wave; kb < blocks;) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        if (kb < blocks) {
          stage(v[d]);
          if (kb + kDepth * kWaves < blocks) load(v[d], kb + kDepth * kWaves);  // the block is in LDS: its registers are free
          multiply(acc);
          kb += kWaves;
        }
      }
    }
    __syncthreads();
    float* sums = (float*)lds;  // [wavefront][block][lane][4], then their sums
#pragma unroll
    for (int i = 0; i < kMB; ++i)
#pragma unroll
      for (int j = 0; j < kNB; ++j) *(f32x4*)(sums + wave * kSums + ((i * kNB + j) * 64 + lane) * 4) = acc[i][j];
    __syncthreads();
    float* total = sums + kWaves * kSums;
    for (int u = (int)threadIdx.x; u < kSums; u += kWaves * 64) {
      float s = sums[u];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s += sums[w * kSums + u];
      total[u] = s;
    }
    __syncthreads();
    // Neighbouring threads take neighbouring columns of a row.
    with_activation(g.activation, [&](auto act) {
      constexpr int kOut = 8 * kNB;
      for (int u = (int)threadIdx.x; u < 16 * kMB * kOut; u += kWaves * 64) {
        const int row = u / kOut, col = u % kOut;
        if (m0 + row >= p.M || col >= left) continue;
        const float* at = total + ((row / 16 * kNB + col / 16) * 64 + (col % 16 / 4) * 16 + row % 16) * 4 + col % 4;
        const float z = at[0], y = at[kNB / 2 * 256];
        if (g.partial) {
          float* to = g.partial + ((int64_t)split * p.M + m0 + row) * (2 * (int64_t)p.N) + n0 + col;
          to[0] = z, to[p.N] = y;
          continue;
        }
        if (g.inner) {
          float slope;
          const float activation = activated<decltype(act)::value, true>(z, slope), d = (float)((const T*)g.grad)[(int64_t)(m0 + row) * g.ld_grad + n0 + col];
          T* inner = (T*)g.inner + (int64_t)(m0 + row) * g.ld_inner + n0 + col;
          inner[0] = to_out<T>(d * y * slope), inner[p.N] = to_out<T>(d * activation);
          continue;
        }
        ((T*)g.out)[(int64_t)(m0 + row) * g.ld_out + n0 + col] = to_out<T>(activated<decltype(act)::value>(z) * y);
        if (g.kept) {
          T* kept = (T*)g.kept + (int64_t)(m0 + row) * g.ld_kept + n0 + col;
          kept[0] = to_out<T>(z), kept[p.N] = to_out<T>(y);
        }
      }
    });
  }
};

template <typename T, int kMB, int kNB, int kWaves, bool kBDeep>
__global__ __launch_bounds__(kWaves * 64, kMB == 1 && kNB == 2 ? 4 : 2) void gated_rows_kernel(GatedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef GatedRows<T, kMB, kNB, kWaves, kBDeep> Tile;
  __shared__ __attribute__((aligned(1024))) char rows_lds[Tile::kLds];
  // An XCD's workgroups have neighbouring columns of a split: of a weight by rows they share lines, and together read stretches of its rows
  // that lie in all of the L2's channels (rows a power of two apart start in the same one).
  const int id = (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds, tiles = a.tiles_m * a.tiles_n;
  if (id >= tiles * a.splits) return;
  const int split = id / tiles, t = id - split * tiles;
  Tile(a, rows_lds).tile(t % a.tiles_m * (16 * kMB), t / a.tiles_m * (8 * kNB), split);
#endif
}

// dx = inner W', the tiles of Product without pairs: of few outputs and a long sum, where the GEMM's kernels, which do not split K, leave CUs without
// work, and of rows that are no whole vectors or operands that reach beyond the GEMM's windows (8192 x 4097 from 8192 545 to 628 us, the GEMM into
// wider rows 510 to 541; 300 x 1001 from 600 9.4 to 12.7, 9.7 to 10.0; 4 x 1001 from 16384 12.9 to 28, 29 to 44).  Sums of splits are added up by
// weight_sum_kernel.  Bound by its turns, as gated_kernel's 128 tiles: 1024 x 2048 from 8192 42 us (the GEMM 62),
// 4142 x 232 from 7952 32 to 35 (70 to 77), 8192 x 128 from 16384 62 (81 to 95).
template <typename T, bool kBDeep>
__global__ __launch_bounds__(512, 2) void input_grad_kernel(InputGradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Product<T, 128, false, kBDeep, false> Tile;
  __shared__ __attribute__((aligned(1024))) char grad_lds[Tile::kLds];
  const int tiles = a.tiles_m * a.tiles_n, item = a.first + (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds;
  if (item >= a.items) return;
  const int split = item / tiles;
  const TileCoord at = tile_coords(item - split * tiles, a.tiles_m, a.tiles_n, a.band);
  const int m0 = at.m * 128, n0 = at.n * 128, first = split * a.blocks_per_split, all = (a.p.K + 63) / 64;
  const int steps = all - first < a.blocks_per_split ? all - first : a.blocks_per_split;
  Tile t(a.p, grad_lds);
  typename Tile::Sums acc;
  Tile::clear(acc);
  if (steps > 0) t.run(acc, m0, n0, first, steps);
#pragma unroll
  for (int i = 0; i < Tile::kRows; ++i)
#pragma unroll
    for (int j = 0; j < Tile::kBlocksN; ++j) {
      const int64_t row = m0 + t.out_row(i);
      const int col = n0 + t.wn * 64 + 16 * j + 4 * (t.lane >> 4);
      if (row < a.p.M && col < a.p.N) {
        if (a.splits > 1)
          put4<float>(acc[i][j], (char*)(a.partial + (int64_t)split * a.p.M * a.ld_partial), row * a.ld_partial + col, a.p.N - col);
        else
          put4<T>(acc[i][j], a.out, row * a.ld_out + col, a.p.N - col);
      }
    }
#endif
}

// What the splits have summed, ascending, and from it what the layer or its gradient gives.  The sums are still in the caches: 13 x 4096 outputs
// from four splits 2.9 us, most of it the launch.
template <typename T, bool kBackward>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int n = a.p.N;
  const int64_t all = (int64_t)a.p.M * n;
  with_activation(a.activation, [&](auto act) {
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (int64_t)gridDim.x * 256) {
      const int64_t row = quotient(u, n), col = u - row * n;
      const float* at = a.partial + row * 2 * n + col;
      float z = at[0], y = at[n];
      for (int split = 1; split < a.splits; ++split) z += at[split * 2 * all], y += at[split * 2 * all + n];
      if constexpr (kBackward) {
        float slope;
        const float activation = activated<decltype(act)::value, true>(z, slope), d = (float)((const T*)a.grad)[row * a.ld_grad + col];
        T* inner = (T*)a.inner + row * a.ld_inner + col;
        inner[0] = to_out<T>(d * y * slope), inner[n] = to_out<T>(d * activation);
      } else {
        ((T*)a.out)[row * a.ld_out + col] = to_out<T>(activated<decltype(act)::value>(z) * y);
        if (a.kept) {
          T* kept = (T*)a.kept + row * a.ld_kept + col;
          kept[0] = to_out<T>(z), kept[n] = to_out<T>(y);
        }
      }
    }
  });
#endif
}

// dg and du from z as it was kept.  Every value is read once; inner may be kept itself.  Bound by memory: 4096 x 4096 bf16 28 us,
// 6.0 TB/s; 8192 x 8192 116, 5.8 (in turns of 8192 workgroups 124).
template <typename T>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int chunks = (a.cols + 7) / 8;
  const int64_t all = (int64_t)a.rows * chunks;
  with_activation(a.activation, [&](auto act) {
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
      const int64_t row = quotient(at, chunks);
      const int col = (int)(at - row * chunks) * 8, left = a.cols - col;
      const typename Eight<T>::Vec dh = Eight<T>::get(a.grad, row * a.ld_grad + col, left), g = Eight<T>::get(a.kept, row * a.ld_kept + col, left),
                                   u = Eight<T>::get(a.kept, row * a.ld_kept + a.cols + col, left);
      typename Eight<T>::Vec dg, du;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float slope;
        const float activation = activated<decltype(act)::value, true>((float)g[e], slope), d = (float)dh[e];
        dg[e] = (T)(d * (float)u[e] * slope);
        du[e] = (T)(d * activation);
      }
      Eight<T>::put(a.inner, row * a.ld_inner + col, left, dg);
      Eight<T>::put(a.inner, row * a.ld_inner + a.cols + col, left, du);
    }
  });
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
