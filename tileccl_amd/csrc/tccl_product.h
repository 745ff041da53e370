// Products of two 16-bit matrices on MFMA tiles, for gfx950, by how each operand lies in memory: the common part of the gated
// layer's projections (tccl_gated.h) and of the weight gradient from an input in full (tccl_weight_full.h), and of the input gradient.
//
//     P[m][n] = sum over k of A(m, k) * B(n, k)
//
// An operand lies by rows (element (i, k) at i * ld + k: k is contiguous) or deep (at k * ld + i: i is).  Rows go through LDS as
// 128 bytes of 64 k each and are read with ds_read_b128; deep operands as 64 k rows, read through the transposing
// ds_read_b64_tr_b16 (within 16 lanes, lane i supplies 4 neighbours of k row i / 4, lane j receives 4 k of column j).  A paired B
// is two matrices that lie `up` bytes apart: of every 64 columns of the tile 32 are the first one's and 32 the same
// columns of the second, so that a lane that has an element of one product has that of the other, too.
//
// global --buffer_load_dwordx4 ... lds--> LDS: lane l's 16 bytes land at base + 16 l, so the swizzles that keep reads off each
// other's banks are applied by choosing what a lane fetches:
//   rows:  chunk c (8 k) of row r in slot c ^ ((r >> 1) & 7)
//   deep:  chunk c (8 columns) of k row k in slot c ^ 4 (k & 3) ^ 2 ((k >> 3) & 1); with k rows of 128 bytes
//          c ^ 2 ((k >> 1) & 1) ^ 4 ((k >> 3) & 1)
// What lies past an operand's window reads as zero; chunks of rows at k >= K are sent there.
#pragma once

#include "tccl_gemm.h"

namespace tccl {

struct ProductArgs {
  const char *a, *b;
  int64_t lda, ldb;  // elements
  int64_t up;        // paired: bytes from the first matrix of B to the second
  int M, N, K;       // N: columns of either matrix of a paired B
};

// Up to three copies in one launch: operands whose rows start anywhere, into rows of whole 16-byte vectors, zero behind their columns.
struct CopyJob {
  const char* from;
  char* to;
  int64_t ld_from, ld_to;  // elements
  int64_t chunks;          // vectors in all
  int cols, per_row;       // columns; vectors of a row
  int first_wg, wgs;       // workgroups that take them
};
struct CopyArgs {
  CopyJob job[3];
  int n;
};

#if defined(__HIPCC__)

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

// kTile x kTile outputs by 2 x kTile / 64 wavefronts, each kTile / 2 x 64.  A 128 tile has two such groups, each of which takes half of the
// steps with stages of its own and ends up with half of the rows of blocks: half the steps one behind the other where tiles are few,
// and no more tiles under way than CUs where they are many.
template <typename T, int kTile, bool kADeep, bool kBDeep, bool kPaired>
struct Product {

  typedef typename Mfma<T>::Vec Vec;
  typedef __attribute__((address_space(3))) void LdsVoid;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 LdsQuad;
  typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
  static constexpr int kWavesN = kTile / 64, kWaves = 2 * kWavesN, kGroups = 8 / kWaves;  // kWaves: of a group
  static constexpr int kStepK = 64;
  static constexpr int kOperand = kTile * 128;  // bytes of an operand in a stage
  static constexpr int kStage = 2 * kOperand, kLds = kGroups * 2 * kStage;
  static constexpr int kBlocksM = kTile / 32, kBlocksN = 4;  // 16 x 16 blocks of a wavefront
  static constexpr int kRows = kBlocksM / kGroups;           // rows of blocks that it ends up with
  static constexpr int kTileN = kPaired ? kTile / 2 : kTile;  // columns of either matrix
  static constexpr int kPitchA = 2 * kTile, kPitchB = 2 * kTileN;  // bytes of a deep operand's k row in a stage

  const ProductArgs& p;
  char *lds, *mine;  // of the workgroup, of the group
  const int lane, group, wave, wm, wn;

  TCCL_D Product(const ProductArgs& args, char* mem)
      : p(args), lds(mem), lane((int)(threadIdx.x & 63)), group(kGroups > 1 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) / kWaves : 0),
        wave(__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) % kWaves), wm(wave / kWavesN), wn(wave % kWavesN) {
    mine = mem + group * 2 * kStage;
  }
  // Row of the tile, of this lane in row i of the blocks that the wavefront ends up with.
  TCCL_D int out_row(int i) const { return wm * (kTile / 2) + 16 * (group * kRows + i) + (lane & 15); }

  // ---- global -> LDS ------------------------------------------------------------------------------
  // A step's operand is fetched in two halves of two pieces (1 KiB, one load) per wavefront.  Rows: half h of a 256 tile's A is rows
  // 64 h .. + 63 of each 128, of the others rows 32 h .. + 31 of each 64 (of a paired B: matrix h).  Deep: k rows 32 h .. + 31
  // (of a paired B: piece i from matrix i).
  static constexpr int row_of(int wave, int h, int i, bool a) {
    return kTile == 256 && a ? (wave >> 2) * 128 + h * 64 + (wave & 3) * 16 + 8 * i : (wave >> 1) * 64 + h * 32 + (wave & 1) * 16 + 8 * i;
  }
  template <int kPitch>
  static TCCL_D int deep_swizzle(int k) {
    return kPitch == 128 ? 2 * ((k >> 1) & 1) ^ 4 * ((k >> 3) & 1) : 4 * (k & 3) ^ 2 * ((k >> 3) & 1);
  }
  struct Side {
    const char* at;     // of the tile and of the step that is loaded next
    int64_t left;       // bytes from there to the end of what may be read
    int64_t step;       // bytes of a step
    uint32_t off[2][2];  // this lane's offsets
    int kt;              // the step
  };
  struct Source {
    Side a, b;
  };

  // Rows: `rows` of them are left from the tile's first on, K elements each.
  template <bool kA>
  TCCL_D void by_rows(Side& s, const char* at, int64_t ld, int rows) const {
    const int kw = (p.K + 7) / 8 * 8;
    s.at = at;
    s.left = ((int64_t)(rows - 1) * ld + kw) * 2;
    s.step = kStepK * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row_of(wave, h, i, kA) + (lane >> 3), kc = (lane & 7) ^ ((row >> 1) & 7);
        const int real = kA || !kPaired ? row : row / 64 * 32 + row % 32;
        s.off[h][i] = (uint32_t)(real * ld * 2 + kc * 16);
      }
  }
  // Deep: `cols` columns are left from the tile's first on.  (Whole vectors are there.)
  template <bool kA>
  TCCL_D void by_depth(Side& s, const char* at, int64_t ld, int cols) const {
    constexpr int kPitch = kA ? kPitchA : kPitchB, kRows = 1024 / kPitch;  // k rows of a piece
    s.at = at;
    s.left = ((int64_t)(p.K - 1) * ld + (cols + 7) / 8 * 8) * 2 + (kA || !kPaired ? 0 : p.up);
    s.step = kStepK * ld * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 32 * h + (kPaired && !kA ? wave : 2 * wave + i) * kRows + lane / (kPitch / 16);
        const int c = lane % (kPitch / 16) ^ deep_swizzle<kPitch>(k);
        s.off[h][i] = (uint32_t)(k * ld * 2 + c * 16 + (kPaired && !kA && i ? p.up : 0));
      }
  }
  TCCL_D Source source(int m0, int n0, int first) const {
    Source s;
    if constexpr (kADeep)
      by_depth<true>(s.a, p.a + (int64_t)m0 * 2, p.lda, p.M - m0);
    else
      by_rows<true>(s.a, p.a + (int64_t)m0 * p.lda * 2, p.lda, p.M - m0);
    if constexpr (kBDeep)
      by_depth<false>(s.b, p.b + (int64_t)n0 * 2, p.ldb, p.N - n0);
    else
      by_rows<false>(s.b, p.b + (int64_t)n0 * p.ldb * 2, p.ldb, p.N - n0);
    start<kADeep>(s.a, first);
    start<kBDeep>(s.b, first);
    return s;
  }
  template <bool kDeep>
  TCCL_D void start(Side& s, int first) const {
    s.at += first * s.step;
    s.left -= first * s.step;
    s.kt = first;
    mask<kDeep>(s);
  }
  static TCCL_D Words4 window(const char* at, int64_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)at;
    Words4 d;
    d[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
    d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    d[2] = __builtin_amdgcn_readfirstlane(bytes > 0xfffffff0ll ? 0xfffffff0u : bytes < 0 ? 0u : (uint32_t)bytes);
    d[3] = 0x00020000u;
    return d;
  }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  // Two loads of 16 bytes per lane, global -> LDS.  Written out because the compiler makes every later read of an LDS array wait for
  // all loads into it.  M0 wants an instruction between its write and the load; a scalar register that a vector instruction has
  // written wants five wait states before a vector memory instruction reads it, which the block spends itself.
  static TCCL_D void copy_pair(char* to0, char* to1, Words4 from, uint32_t off0, uint32_t off1) {
    const uint32_t first = (uint32_t)(uintptr_t)(LdsVoid*)to0, second = (uint32_t)(uintptr_t)(LdsVoid*)to1;
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
        "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds" ::"s"(first), "s"(second), "v"(off0), "v"(off1), "s"(from)
        : "memory", "m0");
  }
#pragma clang diagnostic pop
  static constexpr uint32_t kDead = 0xfffffff0u;  // past the end of every window
  // Half h of A, of B of the source's step into `stage`; behind half 1 the source is the next step's.
  TCCL_D void issue_a(char* stage, Source& s, int h) const {
    char* to0 = stage + (kADeep ? (32 * h + 2 * wave * (1024 / kPitchA)) * kPitchA : row_of(wave, h, 0, true) * 128);
    copy_pair(to0, to0 + 1024, window(s.a.at, s.a.left), s.a.off[h][0], s.a.off[h][1]);
    if (h) advance<kADeep>(s.a);
  }
  TCCL_D void issue_b(char* stage, Source& s, int h) const {
    char* to = stage + kOperand;
    if constexpr (kBDeep && kPaired) {
      to += (32 * h + wave * (1024 / kPitchB)) * kPitchB;
      copy_pair(to, to + kOperand / 2, window(s.b.at, s.b.left), s.b.off[h][0], s.b.off[h][1]);
    } else if constexpr (kBDeep) {
      to += (32 * h + 2 * wave * (1024 / kPitchB)) * kPitchB;
      copy_pair(to, to + 1024, window(s.b.at, s.b.left), s.b.off[h][0], s.b.off[h][1]);
    } else {
      to += row_of(wave, h, 0, false) * 128;
      copy_pair(to, to + 1024, window(s.b.at + (kPaired && h ? p.up : 0), s.b.left), s.b.off[h][0], s.b.off[h][1]);
    }
    if (h) advance<kBDeep>(s.b);
  }
  // Rows, ahead of a step's loads: chunks at k >= K are dead from here on.
  template <bool kDeep>
  TCCL_D void mask(Side& s) const {
    if (kDeep || (s.kt + 1) * kStepK <= p.K) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int kc = (lane & 7) ^ ((4 * i + (lane >> 4)) & 7);
      if (s.kt * kStepK + 8 * kc >= p.K) s.off[0][i] = s.off[1][i] = kDead;
    }
  }
  // Steps past the last one read zeros: deep, nothing is left there; rows, all chunks are dead.
  template <bool kDeep>
  TCCL_D void advance(Side& s) const {
    s.at += s.step, s.left -= s.step;
    ++s.kt;
    mask<kDeep>(s);
  }

  // ---- LDS -> operands ----------------------------------------------------------------------------
  template <int kPitch>
  TCCL_D Vec turned(const char* base, int chunk, int kh) const {
    const int i = lane & 15, g = lane >> 4, t = i >> 2, cq = i & 3;
    const char* q = base + (32 * kh + 8 * g + t) * kPitch + ((chunk + (cq >> 1)) ^ deep_swizzle<kPitch>(8 * g + t)) * 16 + (cq & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)q);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad*)(q + 4 * kPitch));
    return __builtin_bit_cast(Vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  TCCL_D Vec by_row(const char* base, int row, int kh) const {
    const int i = lane & 15;
    return *(const Vec*)(base + (row + i) * 128 + (((4 * kh + (lane >> 4)) ^ ((i >> 1) & 7)) << 4));
  }
  // Block `rb` of 16 rows, of 16 columns of the wavefront's, k block kh (32 k).
  TCCL_D Vec operand_a(const char* stage, int kh, int rb) const {
    const int row = wm * (kTile / 2) + 16 * rb;
    if constexpr (kADeep)
      return turned<kPitchA>(stage, row / 8, kh);
    else
      return by_row(stage, row, kh);
  }
  TCCL_D Vec operand_b(const char* stage, int kh, int cb) const {
    if constexpr (kBDeep && kPaired)
      return turned<kPitchB>(stage + kOperand + (cb >> 1) * (kOperand / 2), wn * 4 + 2 * (cb & 1), kh);
    else if constexpr (kBDeep)
      return turned<kPitchB>(stage + kOperand, wn * 8 + 2 * cb, kh);
    else
      return by_row(stage + kOperand, wn * 64 + 16 * cb, kh);
  }

  typedef f32x4 Sums[kBlocksM][kBlocksN];
  static TCCL_D void clear(Sums& acc) {
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  static TCCL_D void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  }

  template <int kLeft>
  static TCCL_D void wait_loads() {  // until at most kLeft of this wavefront's loads are under way
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
  }

  // The 256 tile.  A step is four phases; in each a wavefront first moves data (two loads, LDS reads) and then multiplies (16 MFMAs,
  // 256 clocks), with a barrier behind either, and wavefronts 4 .. 7 run one such slot behind wavefronts 0 .. 3: of a SIMD's two
  // wavefronts one multiplies while the other moves data.  Either stage is refilled in quarters, as soon as both sides have read one
  // (its last phase, and a phase more), and the waits on loads are counted.
  struct Running {
    Vec a[4], b[2][4];
  };
  TCCL_D void multiply(Sums& acc, const Running& f, int first, int kh) const {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[first + i][j] = Mfma<T>::run16(f.b[kh][j], f.a[i], acc[first + i][j]);
    __builtin_amdgcn_s_setprio(0);
    barrier();
  }
  TCCL_D void read_a(Running& f, const char* stage, int kh, int first) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.a[i] = operand_a(stage, kh, first + i);
  }
  TCCL_D void read_b(Running& f, const char* stage, int kh, int from = 0, int to = 4) const {
#pragma unroll
    for (int j = from; j < to; ++j) f.b[kh][j] = operand_b(stage, kh, j);
  }
  // A by rows: phases are upper rows of the wavefront with k block 0, 1, lower rows with 0, 1.
  //                last read in phase    refilled, with step t + 2, in
  //   B, halves    1                     3, and 0 of the next step
  //   A, upper     1                     1 of the next step
  //   A, lower     3                     2 of the next step
  // Both deep: k block 0 with upper rows, lower, k block 1 with lower, upper.  Halves are k blocks.  Twelve of the
  // transposing reads in each phase: half of a block of B is read in the phase ahead of its own.
  //   B, block 0   0                     2
  //   A, block 0   1                     3
  //   B, block 1   2                     0 of the next step
  //   A, block 1   3                     1 of the next step
  TCCL_D void phases(char* cur, char* nxt, Source& s, Sums& acc, Running& f) const {
    if constexpr (kADeep) {
      issue_b(nxt, s, 1);
      read_b(f, cur, 0, 2, 4);
      read_a(f, cur, 0, 0);
      wait_loads<8>();  // B, block 1 of this step
      multiply(acc, f, 0, 0);
      issue_a(nxt, s, 1);
      read_a(f, cur, 0, 4);
      read_b(f, cur, 1, 0, 2);
      wait_loads<8>();  // A, block 1
      multiply(acc, f, 4, 0);
      issue_b(cur, s, 0);
      read_b(f, cur, 1, 2, 4);
      read_a(f, cur, 1, 4);
      wait_loads<8>();  // B, block 0 of the next step
      multiply(acc, f, 4, 1);
      issue_a(cur, s, 0);
      read_a(f, cur, 1, 0);
      read_b(f, nxt, 0, 0, 2);
      wait_loads<8>();  // A, block 0
      multiply(acc, f, 0, 1);
    } else {
      issue_b(nxt, s, 1);
      read_b(f, cur, 0);
      read_a(f, cur, 0, 0);
      multiply(acc, f, 0, 0);
      issue_a(nxt, s, 0);
      read_b(f, cur, 1);
      read_a(f, cur, 1, 0);
      wait_loads<6>();  // lower rows of this step
      multiply(acc, f, 0, 1);
      issue_a(nxt, s, 1);
      read_a(f, cur, 0, 4);
      multiply(acc, f, 4, 0);
      issue_b(cur, s, 0);
      read_a(f, cur, 1, 4);
      wait_loads<4>();  // B and upper rows of the next step
      multiply(acc, f, 4, 1);
    }
  }

  // The multiplying slot of a 128 tile.
  TCCL_D void whole_step(Sums& acc, const char* cur) const {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      Vec a[kBlocksM], b[kBlocksN];
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) b[j] = operand_b(cur, kh, j);
#pragma unroll
      for (int i = 0; i < kBlocksM; ++i) a[i] = operand_a(cur, kh, i);
#pragma unroll
      for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
        for (int j = 0; j < kBlocksN; ++j) acc[i][j] = Mfma<T>::run16(b[j], a[i], acc[i][j]);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  // acc[0 .. kRows - 1] at the end: lane l has row out_row() and columns 4 (l / 16) .. + 3 of a block.  Steps first .. first + steps - 1; behind
  // them nothing is under way and everybody has left the LDS.
  TCCL_D void run(Sums& acc, int m0, int n0, int first, int steps) const {
    const int turns = kGroups > 1 ? (steps + 1) / 2 : steps, own = group ? steps - turns : turns;
    Source s = source(m0, n0, first + (group ? turns : 0));
    if constexpr (kTile == 256) {
      char* next = lds + kStage;
      issue_b(lds, s, 0);
      if constexpr (kADeep) {
        issue_a(lds, s, 0);
        issue_b(lds, s, 1);
        issue_a(lds, s, 1);
        issue_b(next, s, 0);
        issue_a(next, s, 0);
        wait_loads<8>();
      } else {
        issue_b(lds, s, 1);
        issue_a(lds, s, 0);
        issue_a(lds, s, 1);
        issue_b(next, s, 0);
        wait_loads<4>();
      }
      barrier();
      Running f;
      if constexpr (kADeep) read_b(f, lds, 0, 0, 2);
      if (wave >= 4) barrier();  // one slot behind
      for (int t = 0; t < steps; ++t) phases(lds + (t & 1) * kStage, lds + ((t + 1) & 1) * kStage, s, acc, f);
      if (wave < 4) barrier();
    } else {
      auto load = [&](char* stage) {
        issue_a(stage, s, 0);
        issue_b(stage, s, 0);
        issue_a(stage, s, 1);
        issue_b(stage, s, 1);
      };
      load(mine);
      if (group) barrier();  // one slot behind
      for (int t = 0; t < turns; ++t) {
        const char* cur = mine + (t & 1) * kStage;
        if (t + 1 < turns) {
          load(mine + ((t + 1) & 1) * kStage);
          wait_loads<8>();
        } else {
          wait_loads<0>();
        }
        barrier();
        if (t < own) whole_step(acc, cur);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
      }
      if (!group) barrier();
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    barrier();
    if constexpr (kGroups > 1) join(acc);
  }

  // Each group gives the other half of its rows of blocks away and ends up with the other half in acc[0 .. kRows - 1], group 0 with the first.
  TCCL_D void join(Sums& acc) const {
    constexpr int kHalf = kRows * kBlocksN;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        const f32x4 first = acc[i][j], second = acc[kRows + i][j];  // (values: a choice between places would need them in memory)
        *(f32x4*)(lds + (((group * kWaves + wave) * kHalf + i * kBlocksN + j) * 64 + lane) * 16) = group ? first : second;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        const f32x4 other = *(const f32x4*)(lds + ((((1 - group) * kWaves + wave) * kHalf + i * kBlocksN + j) * 64 + lane) * 16);
        const f32x4 first = acc[i][j] + other, second = other + acc[kRows + i][j];  // group 0's half of the steps first
        acc[i][j] = group ? second : first;
      }
    __syncthreads();
  }
};

// A quotient in 32 bits where that is enough (a 64-bit one is a hundred instructions).
TCCL_D int64_t quotient(int64_t at, int by) { return at >> 32 ? at / by : (int64_t)((uint32_t)at / (uint32_t)by); }

// A thread takes a vector: 16 bytes from anywhere, 16 bytes to a boundary.  12 MB moved in 6 us, 4 of them a launch and a trip to memory.  (A workgroup is one job's: read lane by lane, a job's numbers were a
// chain of trips to memory.)
template <typename T>
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int which = (a.n > 1 && (int)blockIdx.x >= a.job[1].first_wg) + (a.n > 2 && (int)blockIdx.x >= a.job[2].first_wg);
  const CopyJob j = a.job[which];
  for (int64_t u = (int64_t)((int)blockIdx.x - j.first_wg) * 256 + threadIdx.x; u < j.chunks; u += (int64_t)j.wgs * 256) {
    const int64_t row = quotient(u, j.per_row);
    const int col = (int)(u - row * j.per_row) * 8;
    *(typename Eight<T>::Vec*)(j.to + (row * j.ld_to + col) * 2) = Eight<T>::get(j.from, row * j.ld_from + col, j.cols - col);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
