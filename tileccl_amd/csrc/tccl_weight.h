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
  int xcds, span;               // slot -> tile (tile_for_slot)
  int band;                     // tile rows of a band (tile_coords)
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
//
// Three LDS stages of 64 tokens; step t computes from one while the loads of step t + 2 go to the one that step t - 1 has
// left.  The loads are written out (copy_pair), so that the waits on them are counted here.
//
// 256 x 256, eight wavefronts, one workgroup per CU: a step is four phases (row half, token half), in each a wavefront first
// moves data (two loads, LDS reads, the conversions of the phase's operands) and then multiplies (16 MFMAs, 256
// clocks), with a barrier behind either; wavefronts 4..7 run one such slot behind wavefronts 0..3, so that of a SIMD's two
// wavefronts one multiplies while the other moves data.  8-bit operands are read a phase ahead, so that nothing waits for
// LDS within a slot.
// 128 x 128, four wavefronts, two workgroups per CU: one barrier per step; each workgroup's waits are covered by the other.
template <typename T, typename OutT, int kTileH, int kTileN, bool kTransposed>
struct WeightGemm {
  typedef typename Mfma<T>::Vec Vec;
  typedef __attribute__((address_space(3))) void LdsVoid;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 LdsQuad;
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
  static constexpr bool kSides = kTileH == 256;
  static constexpr int kWavesN = kTileN / 64, kWaves = 2 * kWavesN;
  static constexpr int kStepT = 64;                  // tokens of a step
  static constexpr int kRowsX = kTileH * 8;          // bytes of a row block of a stage
  static constexpr int kPitchG = kTileN * 2;         // bytes of a token of a stage
  static constexpr int kStageX = kRowsX * (kStepT / 8), kStageG = kPitchG * kStepT, kStage = kStageX + kStageG;
  static constexpr int kLds = 3 * kStage;
  static constexpr int kBlocksH = kTileH / 32, kBlocksN = 4;  // 16 x 16 blocks of a wavefront
  static_assert(kStageX / 1024 / kWaves == 2 && kStageG / 1024 / kWaves == 4, "loads of a wavefront and step");

  const WeightArgs& a;
  char* lds;
  const int lane, wave, wh, wn;
  int h0, n0;
  uint32_t off_x[2], off_g[2][2];  // this lane's byte offsets within a step

  TCCL_D WeightGemm(const WeightArgs& args, char* mem)
      : a(args), lds(mem), lane((int)(threadIdx.x & 63)), wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))), wh(wave / kWavesN), wn(wave % kWavesN) {}

  static TCCL_D Words4 window(const void* p, int64_t bytes) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    Words4 d;
    d[0] = __builtin_amdgcn_readfirstlane((uint32_t)at);
    d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32) & 0xffffu);
    d[2] = __builtin_amdgcn_readfirstlane(bytes <= 0 ? 0u : bytes > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)bytes);
    d[3] = 0x00020000u;
    return d;
  }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  // Two loads of 16 bytes per lane, global -> LDS, lane l's to `to` + 16 l and `to` + 1024 + 16 l; zero past the window.  Written out
  // because the compiler makes every later read of an LDS array wait for all loads into it.  M0 wants an instruction between
  // its write and the load; a scalar register that a vector instruction has written wants five wait states before a vector memory
  // instruction reads it, which the block spends itself.
  static TCCL_D void copy_pair(char* to, Words4 from, const uint32_t (&off)[2]) {
    const uint32_t first = (uint32_t)(uintptr_t)(LdsVoid*)to, second = first + 1024u;
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
        "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds" ::"s"(first), "s"(second), "v"(off[0]), "v"(off[1]), "s"(from)
        : "memory", "m0");
  }
#pragma clang diagnostic pop

  // Part p of the loads of step t into `stage`: 0 the 8-bit values, 1 and 2 the gradient.  Tokens past the last read as zero:
  // they lie past the end of the window.
  TCCL_D void issue(char* stage, int t, int p) const {
    if (p == 0) {
      const int64_t from = (int64_t)t * (kStepT / 8) * a.value_pitch + (int64_t)h0 * 8;
      copy_pair(stage + 2 * wave * 1024, window(a.values + from, a.row_blocks * a.value_pitch - from), off_x);
    } else {
      const int64_t from = ((int64_t)t * kStepT * a.ld_grad + n0) * 2;
      const int64_t all = ((int64_t)(a.tokens - 1) * a.ld_grad + (a.outputs + 7) / 8 * 8) * 2;
      copy_pair(stage + kStageX + (4 * wave + 2 * (p - 1)) * 1024, window(a.grad + from, all - from), off_g[p - 1]);
    }
  }

  // The scales of the eight row blocks of step t (of the last step, past it).
  TCCL_D u32x2 scales_of(int t) const {
    typedef u32x2 Unaligned __attribute__((aligned(1)));
    int cb = (h0 + wh * (kTileH / 2)) / 128;
    const int last = (int)(a.value_pitch / 1024) - 1;
    cb = cb < last ? cb : last;
    t = t < a.steps ? t : a.steps - 1;
    return *(const Unaligned __attribute__((address_space(1)))*)(a.scales + cb * a.scale_pitch + t * (kStepT / 8));
  }
  // That of the lane's row block in token half h.  (255 is no scale: what lies behind the last row block may be anything.)
  TCCL_D float scale_of(u32x2 s, int h) const {
    const uint32_t e = (s[h] >> (8 * (lane >> 4))) & 255u;
    return __uint_as_float((e < 254u ? e : 254u) << 23);
  }

  // The codes of 16 x 16 x 32 operand b, token half h: the lane's eight tokens of one column.
  TCCL_D u32x2 codes(const char* stage, int h, int b) const {
    const int i = lane & 15, g = lane >> 4;
    const int chunk = (wh * kBlocksH + b) ^ (g & 1);  // 16 columns, 128 bytes
    return *(const u32x2*)(stage + (4 * h + g) * kRowsX + chunk * 128 + i * 8);
  }
  static TCCL_D Vec operand(u32x2 q, float scale) {
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

  static TCCL_D void between() { __builtin_amdgcn_sched_barrier(0); }
  static TCCL_D void barrier() {
    between();
    __builtin_amdgcn_s_barrier();
    between();
    asm volatile("" ::: "memory");
  }
  template <int kLeft>
  static TCCL_D void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
  }

  TCCL_D void multiply(f32x4 (&acc)[kBlocksH][kBlocksN], int first, const Vec (&x)[4], const Vec (&g)[4]) const {
    if (kSides) {
      barrier();
      __builtin_amdgcn_s_setprio(1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[first + i][j] = kTransposed ? Mfma<T>::run16(x[i], g[j], acc[first + i][j]) : Mfma<T>::run16(g[j], x[i], acc[first + i][j]);
    if (kSides) {
      __builtin_amdgcn_s_setprio(0);
      barrier();
    }
  }

  struct Running {
    u32x2 q[2][4];   // codes of this phase and of the next
    Vec g[2][4];     // the gradient's operands of either token half
    u32x2 scales, next_scales;
  };

  // Step t of the large tile.  A stage is last read in phase 2 (codes) and 1 (gradient) of its step and refilled from phase 1 of the next
  // one on: behind two barriers.  The loads of step t + 1 are waited for in phase 2, behind them those of step t + 2 that
  // phases 1 and 2 have issued; they are first read in phase 3.
  TCCL_D void step_sides(const char* cur, const char* nxt, char* far, int t, f32x4 (&acc)[kBlocksH][kBlocksN], Running& f) const {
    const float s0 = scale_of(f.scales, 0), s1 = scale_of(f.scales, 1);
    Vec x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[0][j] = operand_g(cur, 0, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[1][i] = codes(cur, 1, i);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = operand(f.q[0][i], s0);
    multiply(acc, 0, x, f.g[0]);
    issue(far, t + 2, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[1][j] = operand_g(cur, 1, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[0][i] = codes(cur, 0, 4 + i);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = operand(f.q[1][i], s1);
    multiply(acc, 0, x, f.g[1]);
    issue(far, t + 2, 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[1][i] = codes(cur, 1, 4 + i);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = operand(f.q[0][i], s0);
    wait_loads<4>();
    multiply(acc, 4, x, f.g[0]);
    f.scales = f.next_scales;
    f.next_scales = scales_of(t + 2);
    issue(far, t + 2, 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[0][i] = codes(nxt, 0, i);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = operand(f.q[1][i], s1);
    multiply(acc, 4, x, f.g[1]);
  }

  // Step t of the small tile.
  TCCL_D void step_one(const char* cur, char* far, int t, f32x4 (&acc)[kBlocksH][kBlocksN], Running& f) const {
    // The loads of this step have landed (the six of the next may be under way), everybody has left `far`.
    asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    barrier();
    const u32x2 scales = f.scales;
    f.scales = f.next_scales;
    f.next_scales = scales_of(t + 2);
    issue(far, t + 2, 0);
    issue(far, t + 2, 1);
    issue(far, t + 2, 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float s = scale_of(scales, h);
      Vec x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f.g[h][j] = operand_g(cur, h, j);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = operand(codes(cur, h, i), s);
      multiply(acc, 0, x, f.g[h]);
    }
  }

  TCCL_D void run(int tile, int split) {
    const TileCoord at = tile_coords(tile, a.tiles_h, a.tiles_n, a.band);
    h0 = at.m * kTileH, n0 = at.n * kTileN;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int byte = (2 * wave + i) * 1024 + lane * 16, rb = byte / kRowsX, in = byte % kRowsX;
      off_x[i] = (uint32_t)(rb * a.value_pitch + (in ^ (128 * (rb & 1))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int byte = (4 * wave + i) * 1024 + lane * 16, k = byte / kPitchG, slot = byte % kPitchG / 16;
      const int chunk = slot ^ (4 * (k & 3)) ^ (2 * ((k >> 3) & 1));
      off_g[i >> 1][i & 1] = (uint32_t)(k * a.ld_grad * 2 + chunk * 16);
    }
    const int first = split * a.steps_per_split, end = first + a.steps_per_split < a.steps ? first + a.steps_per_split : a.steps;
    f32x4 acc[kBlocksH][kBlocksN];
#pragma unroll
    for (int i = 0; i < kBlocksH; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (first < end) {  // (no tokens: no scales either)
      Running f;
      f.scales = scales_of(first);
      f.next_scales = scales_of(first + 1);
#pragma unroll
      for (int p = 0; p < 3; ++p) issue(lds, first, p);
#pragma unroll
      for (int p = 0; p < 3; ++p) issue(lds + kStage, first + 1, p);
      int cur = 0;
      if (kSides) {
        wait_loads<6>();
        barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) f.q[0][i] = codes(lds, 0, i);
        if (wave >= kWaves / 2) barrier();  // one slot behind
      }
      for (int t = first; t < end; ++t) {
        const int nxt = cur == 2 ? 0 : cur + 1, far = cur == 0 ? 2 : cur - 1;
        if constexpr (kSides)
          step_sides(lds + cur * kStage, lds + nxt * kStage, lds + far * kStage, t, acc, f);
        else
          step_one(lds + cur * kStage, lds + far * kStage, t, acc, f);
        cur = nxt;
      }
      if (kSides && wave < kWaves / 2) barrier();
      wait_loads<0>();
    }
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
__global__ __launch_bounds__(2 * kTileN, 2) void weight_gradient_kernel(WeightArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef WeightGemm<T, OutT, kTileH, kTileN, kTransposed> Gemm;
  __shared__ __attribute__((aligned(1024))) char weight_lds[Gemm::kLds];
  const int tiles = a.tiles_h * a.tiles_n;
  const int slot = (int)blockIdx.x % tiles;
  Gemm gemm(a, weight_lds);
  gemm.run(tile_for_slot(slot, tiles, a.xcds, a.span), (int)blockIdx.x / tiles);
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
