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
  int xcds, per_xcd;            // dies with an L2 of their own; (split, tile) pairs of one
  int staged;                   // `add` is there, fp32, its rows on 16 bytes and within reach: store_staged()
  int band;                     // tile rows of a band (tile_coords)
};

struct WeightSumArgs {
  const float* partial;
  const char* add;
  char* out;
  int64_t ld_partial, ld_add, ld_out, slice;  // slice: elements of one split's partial
  int rows, cols, splits;
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

// Four neighbouring outputs, of which `left` (1 ..) exist.  Rows may start at any element: the accesses say so, and are still one
// instruction (4 x 8001 x 3501: value by value 72 us, so 35).
template <typename OutT>
TCCL_D f32x4 get4(const char* from, int64_t at, int left) {
  typedef OutT Quad __attribute__((ext_vector_type(4), aligned(sizeof(OutT))));
  typedef const Quad __attribute__((address_space(1))) GlobalQuad;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (left >= 4) {
    const Quad o = *(GlobalQuad*)((const OutT*)from + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = (float)o[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) s[e] = (float)((const OutT*)from)[at + e];
  }
  return s;
}
template <typename OutT>
TCCL_D void put4(const f32x4& s, char* to, int64_t at, int left) {
  typedef OutT Quad __attribute__((ext_vector_type(4), aligned(sizeof(OutT))));
  typedef Quad __attribute__((address_space(1))) GlobalQuad;
  if (left >= 4) {
    *(GlobalQuad*)((OutT*)to + at) = (Quad){to_out<OutT>(s[0]), to_out<OutT>(s[1]), to_out<OutT>(s[2]), to_out<OutT>(s[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) ((OutT*)to)[at + e] = to_out<OutT>(s[e]);
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
// kGroups = 2: 128 x 128 with eight wavefronts, of which either half takes half of the tokens with stages of its own; the
// halves' sums meet in LDS.  For few tiles: the work of two workgroups on one tile, without partial sums in memory.
//
// What bounds them.  256 x 256: power (8192 x 4096 x 4096 bf16 207 us, 220 with `add`; 1.41 PFLOP/s in the K loop); what is added and stored
// takes 25 us that one tile per CU cannot hide.  128 x 128, two groups (8192 x 2048 x 2048 69 us): multiplication and operands that
// do not hide each other wholly: 64 us with operands that stay in the L2, 55 with no loads at all, 46 with no multiplication.  Conversions later in
// a half, when their codes are there for certain, change nothing (16384 x 1024 x 512 30.6 -> 31.0).
template <typename T, typename OutT, int kTileH, int kTileN, bool kTransposed, int kGroups>
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
  static constexpr int kLds = kGroups * 3 * kStage;
  static constexpr int kBlocksH = kTileH / 32, kBlocksN = 4;  // 16 x 16 blocks of a wavefront
  static_assert(kStageX / 1024 / kWaves == 2 && kStageG / 1024 / kWaves == 4, "loads of a wavefront and step");

  const WeightArgs& a;
  char* lds;
  const int lane, group, wave, wh, wn;
  int h0, n0;
  uint32_t off_x[2], off_g[2][2];  // this lane's byte offsets within a step

  TCCL_D WeightGemm(const WeightArgs& args, char* mem)
      : a(args), lds(mem + (kGroups > 1 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) / kWaves * 3 * kStage : 0)), lane((int)(threadIdx.x & 63)),
        group(kGroups > 1 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) / kWaves : 0),
        wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) % kWaves), wh(wave / kWavesN), wn(wave % kWavesN) {}

  static TCCL_D Words4 window(const void* p, int64_t bytes) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    Words4 d;
    d[0] = __builtin_amdgcn_readfirstlane((uint32_t)at);
    d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32) & 0xffffu);
    d[2] = __builtin_amdgcn_readfirstlane(bytes > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)bytes);  // (there are always some)
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

  // Where the next step's operands lie, and how many bytes there are from there on.  Steps past the last are the last one again,
  // so that no window begins behind its operand.
  struct Source {
    const uint8_t* x;
    const char* g;
    int64_t left_x, left_g;
    int more;  // steps behind this one
  };
  TCCL_D Source source(int step) const {
    step = step < a.steps ? step : a.steps - 1;
    const int64_t from_x = (int64_t)step * (kStepT / 8) * a.value_pitch + (int64_t)h0 * 8, from_g = ((int64_t)step * kStepT * a.ld_grad + n0) * 2;
    return Source{a.values + from_x, a.grad + from_g, a.row_blocks * a.value_pitch - from_x,
                  ((int64_t)(a.tokens - 1) * a.ld_grad + (a.outputs + 7) / 8 * 8) * 2 - from_g, a.steps - 1 - step};
  }
  // Part p of the loads of a step into `stage`: 0 the 8-bit values, 1 and 2 the gradient; behind part 2 the source is the next
  // step's.  Tokens past the last read as zero: they lie past the end of the window.
  TCCL_D void issue(char* stage, Source& s, int p) const {
    if (p == 0) {
      copy_pair(stage + 2 * wave * 1024, window(s.x, s.left_x), off_x);
    } else {
      copy_pair(stage + kStageX + (4 * wave + 2 * (p - 1)) * 1024, window(s.g, s.left_g), off_g[p - 1]);
      if (p == 2) {
        const int64_t step_x = s.more > 0 ? (kStepT / 8) * a.value_pitch : 0, step_g = s.more > 0 ? kStepT * 2 * a.ld_grad : 0;
        s.x += step_x, s.left_x -= step_x;
        s.g += step_g, s.left_g -= step_g;
        --s.more;
      }
    }
  }

  // The scales of the wavefront's column block for kScaleSteps steps from `first` on: lane l has those of row blocks 16 l ..
  // 16 l + 15.  `first` is even: a step has 8 row blocks, and a 16-byte read from an odd one would end 8 bytes behind the row, for
  // the last column block behind the scales.  One load for 8192 tokens: an ordinary load in every step would be waited for with everything behind it, the copies
  // of the next stages (the compiler does not count those).
  static constexpr int kScaleSteps = 128;
  TCCL_D Words4 scales_from(int first) const {
    typedef Words4 Unaligned __attribute__((aligned(1)));  // (the scales' address may be any)
    typedef const Unaligned __attribute__((address_space(1))) Global;
    int cb = (h0 + wh * (kTileH / 2)) / 128;
    const int last = (int)(a.value_pitch / 1024) - 1;
    cb = cb < last ? cb : last;
    const int64_t at = (int64_t)first * (kStepT / 8) + 16 * lane;
    Words4 s = {0, 0, 0, 0};
    if (at < a.scale_pitch) s = *(Global*)(a.scales + cb * a.scale_pitch + at);
    asm volatile("" : "+v"(s));  // waited for here, not in the loop
    return s;
  }
  // That of the lane's row block in token half h of the step that is `n` steps behind the first.  (255 is no scale: what lies
  // behind the last row block may be anything.)
  TCCL_D float scale_of(const Words4& s, int n, int h) const {
    const uint32_t even = __builtin_amdgcn_readlane(s[h], n >> 1), odd = __builtin_amdgcn_readlane(s[2 + h], n >> 1);
    const uint32_t e = ((n & 1 ? odd : even) >> (8 * (lane >> 4))) & 255u;
    return __uint_as_float((e < 254u ? e : 254u) << 23);
  }

  // The codes of 16 x 16 x 32 operand b, token half h: the lane's eight tokens of one column.
  TCCL_D u32x2 codes(const char* stage, int h, int b) const {
    const int i = lane & 15, g = lane >> 4;
    const int chunk = (wh * kBlocksH + b) ^ (g & 1);  // 16 columns, 128 bytes
    return *(const u32x2*)(stage + (4 * h + g) * kRowsX + chunk * 128 + i * 8);
  }
  // Dword w (tokens 2w, 2w + 1) of the operand that codes are converted to.
  static TCCL_D uint32_t converted(u32x2 q, int w, float scale) {
    return __builtin_bit_cast(uint32_t, w & 1 ? FromHeld<T>::template pair<true>(q[w >> 1], scale) : FromHeld<T>::template pair<false>(q[w >> 1], scale));
  }
  static TCCL_D Words4 operand(u32x2 q, float scale) { return (Words4){converted(q, 0, scale), converted(q, 1, scale), converted(q, 2, scale), converted(q, 3, scale)}; }
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

  static TCCL_D f32x4 product(Words4 x, Vec g, f32x4 c) {
    const Vec v = __builtin_bit_cast(Vec, x);
    return kTransposed ? Mfma<T>::run16(v, g, c) : Mfma<T>::run16(g, v, c);
  }

  struct Running {
    u32x2 q[4];      // codes of the next phase
    Words4 x[2][4];  // 8-bit operands, converted, of this phase and the next
    Vec g[2][4];     // the gradient's operands of either token half
    Words4 scales;   // from step scales_at on
    int scales_at;
  };

  // 16 MFMAs from operand sets kX and kG, behind each the conversion of two values of the next operands.
  template <int kX, int kG>
  TCCL_D void multiply(f32x4 (&acc)[kBlocksH][kBlocksN], int first, Running& f, float next_scale) const {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[first + i][j] = product(f.x[kX][i], f.g[kG][j], acc[first + i][j]);
        f.x[1 - kX][j][i] = converted(f.q[j], i, next_scale);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      }
    __builtin_amdgcn_s_setprio(0);
  }
  // The multiplying slot of phase `kPhase` of the large tile.
  template <int kPhase>
  TCCL_D void slot(f32x4 (&acc)[kBlocksH][kBlocksN], Running& f, float next_scale) const {
    barrier();
    multiply<kPhase & 1, kPhase & 1>(acc, kPhase < 2 ? 0 : 4, f, next_scale);
    barrier();
  }

  // Step t of the large tile; `next`: the scale of the next step's first half.  A stage is last read in phase 2 (codes) and 1
  // (gradient) of its step and refilled from phase 1 of the next one on: behind two barriers.  The loads of step t + 1 are waited for in
  // phase 2, behind them those of step t + 2 that phases 1 and 2 have issued; they are first read in phase 3.
  TCCL_D void step_sides(const char* cur, const char* nxt, char* far, Source& src, float s0, float s1, float next, f32x4 (&acc)[kBlocksH][kBlocksN], Running& f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(cur, 1, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[0][j] = operand_g(cur, 0, j);
    slot<0>(acc, f, s1);
    issue(far, src, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(cur, 0, 4 + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[1][j] = operand_g(cur, 1, j);
    slot<1>(acc, f, s0);
    issue(far, src, 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(cur, 1, 4 + i);
    wait_loads<4>();
    slot<2>(acc, f, s1);
    issue(far, src, 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(nxt, 0, i);
    slot<3>(acc, f, next);
  }

  // A step of the small tile, whose first half's operands are there.  Either half reads the next one's while it multiplies; the loads of
  // the next step are waited for in between, and those of the step after the next two go to the stage that everybody has left then.
  // `live`: false where the other group has a step more.
  TCCL_D void step_one(char* cur, const char* nxt, Source& src, float s1, float next, f32x4 (&acc)[kBlocksH][kBlocksN], Running& f, bool live) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(cur, 1, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[1][j] = operand_g(cur, 1, j);
    between();
    if (kGroups == 1 || live) multiply<0, 0>(acc, 0, f, s1);
    between();
    asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) f.q[i] = codes(nxt, 0, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[0][j] = operand_g(nxt, 0, j);
#pragma unroll
    for (int p = 0; p < 3; ++p) issue(cur, src, p);
    between();
    if (kGroups == 1 || live) multiply<1, 1>(acc, 0, f, next);
    between();
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
    int first = split * a.steps_per_split, end = first + a.steps_per_split < a.steps ? first + a.steps_per_split : a.steps;
    int turns = end - first;
    if (kGroups > 1) {  // either group takes as many turns; the second one may have a step fewer
      turns = (end - first + 1) / 2;
      first += group * turns;
      end = group ? end : first + turns;
    }
    f32x4 acc[kBlocksH][kBlocksN];
#pragma unroll
    for (int i = 0; i < kBlocksH; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (turns > 0) {  // (no tokens: no scales either)
      Running f;
      Source src = source(first);
#pragma unroll
      for (int p = 0; p < 3; ++p) issue(lds, src, p);
#pragma unroll
      for (int p = 0; p < 3; ++p) issue(lds + kStage, src, p);
      if (!kSides) {
#pragma unroll
        for (int p = 0; p < 3; ++p) issue(lds + 2 * kStage, src, p);
      }
      f.scales_at = first & ~1;
      f.scales = scales_from(f.scales_at);
      int cur = 0;
      float s0 = scale_of(f.scales, first - f.scales_at, 0);
      wait_loads<kSides ? 6 : 12>();
      barrier();
      if (!kSides) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f.x[0][i] = operand(codes(lds, 0, i), s0);
#pragma unroll
        for (int j = 0; j < 4; ++j) f.g[0][j] = operand_g(lds, 0, j);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f.x[0][i] = operand(codes(lds, 0, i), s0);
        if (wave >= kWaves / 2) barrier();  // one slot behind
      }
      for (int t = first; t < first + turns; ++t) {
        const int nxt = cur == 2 ? 0 : cur + 1, far = cur == 0 ? 2 : cur - 1;
        const float s1 = scale_of(f.scales, t - f.scales_at, 1);
        if (t + 1 - f.scales_at == kScaleSteps) {
          f.scales = scales_from(t + 1);
          f.scales_at = t + 1;
        }
        const float next = scale_of(f.scales, t + 1 - f.scales_at, 0);
        if constexpr (kSides)
          step_sides(lds + cur * kStage, lds + nxt * kStage, lds + far * kStage, src, s0, s1, next, acc, f);
        else
          step_one(lds + cur * kStage, lds + nxt * kStage, src, s1, next, acc, f, t < end);
        s0 = next;
        cur = nxt;
      }
      if (kSides && wave < kWaves / 2) barrier();
      wait_loads<0>();
    }
    if constexpr (kGroups > 1) {
      join(acc);
      store<kBlocksH / 2>(acc, split, group * (kBlocksH / 2));
      return;
    }
    if constexpr (kSides && sizeof(OutT) == 4)
      if (a.staged && h0 + kTileH <= a.cols && n0 + kTileN <= a.outputs) return store_staged(acc);
    store<kBlocksH>(acc, split, 0);
  }

  // A whole 256 x 256 tile of fp32 on top of `add`: the tile's rows of `add` come through LDS, 128 of them (1 KiB each, one
  // load) in either of two rounds; round 1 is on its way while round 0 is added and stored.  Round r has the rows of the
  // wavefronts' blocks i (transposed: j) of half r.  16-byte chunk c of row k lies in slot c ^ (k % 16), which spreads the
  // 16 rows that a read takes over the banks.  Read block by block, 64 bytes of 16 rows at a time, 64 MiB that are not in a
  // cache cost 8192 x 4096 x 4096 34 us.
  TCCL_D void store_staged(f32x4 (&acc)[kBlocksH][kBlocksN]) const {
    const int i16 = lane & 15, g = lane >> 4;
    const int row0 = kTransposed ? n0 : h0, col0 = kTransposed ? h0 : n0;
    constexpr int kPart = kTransposed ? 32 : 64;  // consecutive rows of a round
    const Words4 from = window((const float*)a.add + row0 * a.ld_add + col0, 0xfffffff0ll);
    auto fetch = [&](int r) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        uint32_t off[2];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int k = 16 * wave + 2 * p + o, row = k / kPart * (2 * kPart) + r * kPart + k % kPart;
          off[o] = (uint32_t)(row * a.ld_add * 4) + (uint32_t)((lane ^ (k & 15)) * 16);
        }
        copy_pair(lds + (16 * wave + 2 * p) * 1024, from, off);
      }
    };
    constexpr int kI = kTransposed ? kBlocksH : 4, kJ = kTransposed ? 2 : 4;  // blocks of a round
    barrier();  // everybody has read the last stage
    fetch(0);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      f32x4 more[kI][kJ];
      wait_loads<0>();
      barrier();
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int k = (kTransposed ? wn * 32 + 16 * j : wh * 64 + 16 * i) + i16;
          const int c = (kTransposed ? wh * 32 + 4 * i : wn * 16 + 4 * j) + g;
          more[i][j] = *(const f32x4*)(lds + k * 1024 + ((c ^ i16) * 16));
        }
      if (r == 0) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        fetch(1);
      }
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int bi = kTransposed ? i : 4 * r + i, bj = kTransposed ? 2 * r + j : j;
          const int h = h0 + wh * (kTileH / 2) + 16 * bi, n = n0 + wn * 64 + 16 * bj;
          const int64_t row = (kTransposed ? n : h) + i16, col = (kTransposed ? h : n) + 4 * g;
          put4<float>(acc[bi][bj] + more[i][j], a.out, row * a.ld_out + col, 4);
        }
    }
  }

  // The two groups' sums: each gives the other half of its rows of blocks away and has the other half, group 0 the first.
  TCCL_D void join(f32x4 (&acc)[kBlocksH][kBlocksN]) const {
    char* base = lds - group * 3 * kStage;
    constexpr int kHalf = kBlocksH / 2 * kBlocksN;
    barrier();  // everybody has read the last stages
#pragma unroll
    for (int i = 0; i < kBlocksH / 2; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j)
        *(f32x4*)(base + (((group * kWaves + wave) * kHalf + i * kBlocksN + j) * 64 + lane) * 16) = group ? acc[i][j] : acc[kBlocksH / 2 + i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlocksH / 2; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        const f32x4 other = *(const f32x4*)(base + ((((1 - group) * kWaves + wave) * kHalf + i * kBlocksN + j) * 64 + lane) * 16);
        // (group 0's half of the tokens first, whoever adds)
        acc[i][j] = group ? other + acc[kBlocksH / 2 + i][j] : acc[i][j] + other;
      }
  }

  // Rows of blocks 0 .. kRows - 1 of `acc`, which are `from` .. of the wavefront's.  Lane l has out-row l % 16 of a block and 4
  // neighbouring columns 4 * (l / 16) .. of the row.  What is added is read for several rows of blocks at once: one trip to memory
  // for each half of a wavefront's outputs instead of one for each few.
  template <int kRows>
  TCCL_D void store(f32x4 (&acc)[kBlocksH][kBlocksN], int split, int from) const {
    const int i16 = lane & 15, g = lane >> 4;
    const int rows = kTransposed ? a.outputs : a.cols, cols = kTransposed ? a.cols : a.outputs;
    constexpr int kAtOnce = kRows < 4 ? kRows : 4;
#pragma unroll
    for (int half = 0; half < kRows; half += kAtOnce) {
      const int h1 = h0 + wh * (kTileH / 2) + 16 * (from + half), n1 = n0 + wn * 64;
      if (a.splits == 1 && a.add) {
        f32x4 more[kAtOnce][kBlocksN];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int j = 0; j < kBlocksN; ++j) {
            const int h = h1 + 16 * i, n = n1 + 16 * j, row = kTransposed ? n + i16 : h + i16, col = (kTransposed ? h : n) + 4 * g;
            more[i][j] = row < rows && col < cols ? get4<OutT>(a.add, row * a.ld_add + col, cols - col) : (f32x4){0.f, 0.f, 0.f, 0.f};
          }
        between();
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int j = 0; j < kBlocksN; ++j) acc[half + i][j] += more[i][j];
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < kBlocksN; ++j) {
          const int h = h1 + 16 * i, n = n1 + 16 * j, row = kTransposed ? n + i16 : h + i16, col = (kTransposed ? h : n) + 4 * g;
          if (row < rows && col < cols) {
            if (a.splits > 1)
              put4<float>(acc[half + i][j], (char*)(a.partial + (int64_t)split * rows * a.ld_partial), row * a.ld_partial + col, cols - col);
            else
              put4<OutT>(acc[half + i][j], a.out, row * a.ld_out + col, cols - col);
          }
        }
      between();
    }
  }
};

template <typename T, typename OutT, int kTileH, int kTileN, bool kTransposed, int kGroups>
__global__ __launch_bounds__(2 * kTileN * kGroups, 2) void weight_gradient_kernel(WeightArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef WeightGemm<T, OutT, kTileH, kTileN, kTransposed, kGroups> Gemm;
  __shared__ __attribute__((aligned(1024))) char weight_lds[Gemm::kLds];
  // Workgroups go to the XCDs in turn.  XCD x takes a run of the (split, tile) pairs: the tiles of a split, neighbours of each
  // other, which read the same rows of the operands, find them in one L2 (16384 x 1024 x 512: 30.9 -> 29.3 us).
  const int tiles = a.tiles_h * a.tiles_n, item = (int)blockIdx.x % a.xcds * a.per_xcd + (int)blockIdx.x / a.xcds;
  if (item >= tiles * a.splits) return;
  Gemm gemm(a, weight_lds);
  gemm.run(item % tiles, item / tiles);
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
    for (int first = 1; first < a.splits; first += 8) {  // eight on their way at a time (16384 x 256 x 256: 24 -> 20 us)
      f32x4 more[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) more[k] = first + k < a.splits ? *(const f32x4*)(p + (first + k) * a.slice) : (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (first + k < a.splits) s += more[k];
    }
    if (a.add) s += get4<OutT>(a.add, row * a.ld_add + col, a.cols - col);
    put4<OutT>(s, a.out, row * a.ld_out + col, a.cols - col);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
