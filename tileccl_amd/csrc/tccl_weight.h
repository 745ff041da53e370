// Weight gradient of a linear layer from its input in 8 bits, for gfx950:
//     W[h][n] = sum over tokens t of x[t][h] * grad[t][n] (+ add[h][n]),   x = q * 2^e.
//
// Both operands lie with the summed index outermost.  The 8-bit layout (tccl_norm.h) holds the 8 consecutive tokens that
// a lane of v_mfma_f32_16x16x32 takes of a column as 8 contiguous bytes: a plain 8-byte LDS read, four conversions with
// the scale inside (v_cvt_scalef32_pk_bf16_fp8: exact, a held value is exact in the 16-bit type) and the operand is
// there, with half the LDS bytes of a 16-bit one.  The gradient comes out of LDS through the transposing reads.
#pragma once

#include "tccl_gemm.h"

namespace tccl {

struct WeightArgs {
  const uint8_t *values, *scales;
  const char* grad;
  const char* add;
  char* out;
  float* partial;               // [split][rows of out][ld_partial], where the tokens are split
  int64_t value_pitch, scale_pitch;
  int64_t ld_grad, ld_add, ld_out;  // elements
  int64_t ld_partial;
  int tokens, cols, outputs;
  int row_blocks;               // ceil(tokens / 8)
  int tiles_h, tiles_n;
  int steps, splits;            // steps of 64 tokens; a split takes steps_per_split of them
  int steps_per_split;
  int wide;                     // rows of out and add start on four elements
};

struct WeightSumArgs {
  const float* partial;
  const char* add;
  char* out;
  int64_t ld_partial, ld_add, ld_out, slice;  // slice: elements of one split's partial
  int rows, cols, splits, wide;
};

#if defined(__HIPCC__)

template <typename T>
struct FromHeld;
template <>
struct FromHeld<__bf16> {
  typedef __bf16 Pair __attribute__((ext_vector_type(2)));
  template <bool kHigh>
  static TCCL_D Pair pair(uint32_t q, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)q, scale, kHigh); }
};
template <>
struct FromHeld<_Float16> {
  typedef _Float16 Pair __attribute__((ext_vector_type(2)));
  template <bool kHigh>
  static TCCL_D Pair pair(uint32_t q, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)q, scale, kHigh); }
};

// Four neighbouring outputs; `left` (1 ..) columns exist from the first on.
template <typename OutT>
TCCL_D void put4(const f32x4& v, const char* add, int64_t add_at, char* out, int64_t out_at, int left, bool wide) {
  typedef OutT Quad __attribute__((ext_vector_type(4)));
  f32x4 s = v;
  if (wide && left >= 4) {
    if (add) {
      const Quad o = *(const Quad*)((const OutT*)add + add_at);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += (float)o[e];
    }
    *(Quad*)((OutT*)out + out_at) = (Quad){to_out<OutT>(s[0]), to_out<OutT>(s[1]), to_out<OutT>(s[2]), to_out<OutT>(s[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        if (add) s[e] += (float)((const OutT*)add)[add_at + e];
        ((OutT*)out)[out_at + e] = to_out<OutT>(s[e]);
      }
  }
}

// kTileH x kTileN outputs, wavefronts 2 x kTileN / 64, each kTileH / 2 x 64.
template <typename T, typename OutT, int kTileH, int kTileN, bool kTransposed>
struct WeightGemm {
  typedef typename Mfma<T>::Vec Vec;
  typedef __attribute__((address_space(3))) void LdsVoid;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 LdsQuad;
  static constexpr int kWavesN = kTileN / 64, kWaves = 2 * kWavesN, kThreadsW = 64 * kWaves;
  static constexpr int kStepT = 64;                  // tokens of a step
  static constexpr int kRowsX = kTileH * 8;          // bytes of a row block of a stage
  static constexpr int kPitchG = kTileN * 2;         // bytes of a token of a stage
  static constexpr int kStageX = kRowsX * (kStepT / 8), kStageG = kPitchG * kStepT, kStage = kStageX + kStageG;
  static constexpr int kStages = 3;
  static constexpr int kLds = kStages * kStage;
  static constexpr int kLoadsX = kStageX / 1024 / kWaves, kLoadsG = kStageG / 1024 / kWaves, kLoads = kLoadsX + kLoadsG;
  static constexpr int kBlocksH = kTileH / 32, kBlocksN = 4;  // 16 x 16 blocks of a wavefront

  const WeightArgs& a;
  char* lds;
  const int lane, wave, wh, wn;
  int h0, n0;
  uint32_t off_x[kLoadsX], off_g[kLoadsG];

  TCCL_D WeightGemm(const WeightArgs& args, char* mem)
      : a(args), lds(mem), lane((int)(threadIdx.x & 63)), wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))), wh(wave / kWavesN), wn(wave % kWavesN) {}

  static TCCL_D uint32_t clamped(int64_t bytes) { return bytes <= 0 ? 0u : bytes > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)bytes; }

  // The loads of step `t` into a stage.  Tokens past the last read as zero: they lie past the end of the window.
  TCCL_D void issue(char* stage, int t) const {
    const int64_t from_x = (int64_t)t * (kStepT / 8) * a.value_pitch + (int64_t)h0 * 8;
    const int64_t from_g = ((int64_t)t * kStepT * a.ld_grad + n0) * 2;
    const int64_t all_x = a.row_blocks * a.value_pitch, all_g = ((int64_t)(a.tokens - 1) * a.ld_grad + (a.outputs + 7) / 8 * 8) * 2;
    const __amdgpu_buffer_rsrc_t x = __builtin_amdgcn_make_buffer_rsrc((void*)(a.values + from_x), 0, clamped(all_x - from_x), 0x00020000);
    const __amdgpu_buffer_rsrc_t g = __builtin_amdgcn_make_buffer_rsrc((void*)(a.grad + from_g), 0, clamped(all_g - from_g), 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(x, (LdsVoid*)(stage + (kLoadsX * wave + i) * 1024), 16, off_x[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoadsG; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(g, (LdsVoid*)(stage + kStageX + (kLoadsG * wave + i) * 1024), 16, off_g[i], 0, 0, 0);
  }

  // The scale of the lane's row block of step t, half h (32 tokens).
  TCCL_D uint32_t scale_bits(int t, int h) const {
    int rb = t * (kStepT / 8) + 4 * h + (lane >> 4);
    rb = rb < a.row_blocks ? rb : a.row_blocks - 1;
    int cb = (h0 + wh * (kTileH / 2)) / 128;
    const int last = (int)(a.value_pitch / 1024) - 1;
    cb = cb < last ? cb : last;
    return a.scales[cb * a.scale_pitch + rb];
  }

  TCCL_D Vec operand_x(const char* stage, int h, int b, float scale) const {
    const int i = lane & 15, g = lane >> 4, rb = 4 * h + g;
    const int chunk = (wh * kBlocksH + b) ^ (rb & 1);  // 16 columns, 128 bytes
    const u32x2 q = *(const u32x2*)(stage + rb * kRowsX + chunk * 128 + i * 8);
    typedef typename FromHeld<T>::Pair Pair;
    const Pair p0 = FromHeld<T>::template pair<false>(q[0], scale), p1 = FromHeld<T>::template pair<true>(q[0], scale);
    const Pair p2 = FromHeld<T>::template pair<false>(q[1], scale), p3 = FromHeld<T>::template pair<true>(q[1], scale);
    return (Vec){p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
  }
  TCCL_D Vec operand_g(const char* stage, int h, int b) const {
    const int i = lane & 15, g = lane >> 4, t = i >> 2, cq = i & 3;
    const int chunk = (wn * 8 + 2 * b + (cq >> 1)) ^ (4 * t) ^ (2 * (g & 1));
    const char* p = stage + kStageX + (32 * h + 8 * g + t) * kPitchG + chunk * 16 + (cq & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(p + 4 * kPitchG));
    return __builtin_bit_cast(Vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

  TCCL_D void run(int tile, int split) {
    h0 = (tile / a.tiles_n) * kTileH, n0 = (tile % a.tiles_n) * kTileN;
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i) {
      const int byte = (kLoadsX * wave + i) * 1024 + lane * 16, rb = byte / kRowsX, at = byte % kRowsX;
      off_x[i] = (uint32_t)(rb * a.value_pitch + (at ^ (128 * (rb & 1))));
    }
#pragma unroll
    for (int i = 0; i < kLoadsG; ++i) {
      const int byte = (kLoadsG * wave + i) * 1024 + lane * 16, k = byte / kPitchG, slot = byte % kPitchG / 16;
      const int chunk = slot ^ (4 * (k & 3)) ^ (2 * ((k >> 3) & 1));
      off_g[i] = (uint32_t)(k * a.ld_grad * 2 + chunk * 16);
    }
    const int first = split * a.steps_per_split, end = first + a.steps_per_split < a.steps ? first + a.steps_per_split : a.steps;
    f32x4 acc[kBlocksH][kBlocksN];
#pragma unroll
    for (int i = 0; i < kBlocksH; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    uint32_t bits[2] = {0, 0}, next_bits[2] = {0, 0};
    if (first < end) {  // no tokens: no scales either
      bits[0] = scale_bits(first, 0), bits[1] = scale_bits(first, 1);
      issue(lds, first);
      issue(lds + kStage, first + 1);
    }
    int cur = 0;
    for (int t = first; t < end; ++t) {
      // The loads of this step have landed (those of the next may be under way), everybody has left the stage
      // that is filled next.
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int far = cur == 0 ? 2 : cur - 1;
      next_bits[0] = scale_bits(t + 1, 0), next_bits[1] = scale_bits(t + 1, 1);
      issue(lds + far * kStage, t + 2);
      const char* stage = lds + cur * kStage;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float scale = __uint_as_float(bits[h] << 23);
        Vec g[kBlocksN];
#pragma unroll
        for (int j = 0; j < kBlocksN; ++j) g[j] = operand_g(stage, h, j);
#pragma unroll
        for (int i = 0; i < kBlocksH; ++i) {
          const Vec x = operand_x(stage, h, i, scale);
#pragma unroll
          for (int j = 0; j < kBlocksN; ++j) acc[i][j] = kTransposed ? Mfma<T>::run16(x, g[j], acc[i][j]) : Mfma<T>::run16(g[j], x, acc[i][j]);
        }
      }
      bits[0] = next_bits[0], bits[1] = next_bits[1];
      cur = cur == 2 ? 0 : cur + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    store(acc, split);
  }

  // Lane l has out-row i % 16 of a block and 4 neighbouring columns 4 * (l / 16) .. of the row.
  TCCL_D void store(const f32x4 (&acc)[kBlocksH][kBlocksN], int split) const {
    const int i16 = lane & 15, g = lane >> 4;
    const int rows = kTransposed ? a.outputs : a.cols, cols = kTransposed ? a.cols : a.outputs;
#pragma unroll
    for (int i = 0; i < kBlocksH; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        const int h = h0 + wh * (kTileH / 2) + 16 * i, n = n0 + wn * 64 + 16 * j;
        const int row = kTransposed ? n + i16 : h + i16, col = (kTransposed ? h : n) + 4 * g;
        if (row < rows && col < cols) store4(acc[i][j], row, col, cols - col, split, rows);
      }
  }
  TCCL_D void store4(f32x4 v, int row, int col, int left, int split, int rows) const {
    if (a.splits > 1)
      put4<float>(v, nullptr, 0, (char*)(a.partial + (int64_t)split * rows * a.ld_partial), row * a.ld_partial + col, left, true);
    else
      put4<OutT>(v, a.add, row * a.ld_add + col, a.out, row * a.ld_out + col, left, a.wide);
  }
};

template <typename T, typename OutT, int kTileH, int kTileN, bool kTransposed>
__global__ __launch_bounds__(2 * kTileN, 1) void weight_gradient_kernel(WeightArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef WeightGemm<T, OutT, kTileH, kTileN, kTransposed> Gemm;
  __shared__ __attribute__((aligned(1024))) char weight_lds[Gemm::kLds];
  const int tiles = a.tiles_h * a.tiles_n;
  const int slot = (int)blockIdx.x;
  Gemm gemm(a, weight_lds);
  gemm.run(slot % tiles, slot / tiles);
#endif
}

// out = sum over splits of the partials, ascending, plus add.
template <typename OutT>
__global__ __launch_bounds__(256) void weight_sum_kernel(WeightSumArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int quads = (a.cols + 3) / 4;
  const int64_t all = (int64_t)a.rows * quads;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (int64_t)gridDim.x * 256) {
    const int row = (int)(u / quads), col = (int)(u % quads) * 4;
    const float* p = a.partial + row * a.ld_partial + col;
    f32x4 s = *(const f32x4*)p;
    for (int k = 1; k < a.splits; ++k) s += *(const f32x4*)(p + k * a.slice);
    put4<OutT>(s, a.add, row * a.ld_add + col, a.out, row * a.ld_out + col, a.cols - col, a.wide);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
