// Layer norm, its gradients, and activations held in 8 bits, for gfx950.
//
// Mathematics.  Forward, for a row s of H values (s = x, or x + residual rounded to x's type):
//     mean = sum s / H,  var = sum (s - mean)^2 / H,  rstd = 1 / sqrt(var + eps),  y = (s - mean) rstd gamma + beta.
// Backward, with xh = (s - mean) rstd and g = dy gamma:
//     dx = rstd (g - sum g / H - xh sum(g xh) / H) [+ the gradient that reaches s past the norm],
//     dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy.
// 8-bit values: blocks of 8 rows x 128 columns with a scale 2^e; q = e4m3(s / 2^e), to nearest even.  The scale is a
// power of two: division by it and the value q 2^e are exact (also as a 16-bit float), and a floating 8-bit type gains
// no precision from a finer one.
//
// Layout of the work.  A group of W wavefronts holds R whole rows in registers: a thread has vectors of 8 columns, 16
// (fp32: 32) bytes of each row, NV of them 512 W columns apart.  Every value is read once; the sums of a row meet in LDS.
// The variance is summed around a mean, never as a difference of sums: each wavefront takes its own mean and sum of
// squares around it, and the W pairs are joined as M2 = sum M2_w + n_w (mean_w - mean)^2, which needs one exchange and
// one barrier instead of two.  Workgroups stay and walk over the rows, with gamma, beta and the column sums of the backward
// pass in registers; the column sums of all groups are added by a second launch in a fixed order, so that results
// do not depend on which workgroup comes first.
//
// What bounds them: memory where there are many rows (bf16: 8192 x 4096 forward 24.6 us, 5.4 TB/s with the launch, where a copy reaches 6.45
// without; 16384 x 4096 backward with a residual's gradient 99 us, 5.4; 16384 x 4096 to 8 bits 34 us, back 29), a launch and one or two trips to
// memory where there are few (16 x 4096 6.2 us, of which an empty launch is 3.5).
//
// 8 rows x 8 columns of a thread are also the unit of the 8-bit layout: values lie as [row block][column][row in block], so a
// thread's patch is 64 contiguous bytes, two neighbouring rows of a column go into one conversion, and the weight gradient
// finds the 8 consecutive rows that a lane of a matrix instruction takes as 8 contiguous bytes, with no transposition.
// 16 neighbouring lanes hold a block of 128 columns, which is one row of the data-parallel primitives.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "tccl_device.h"

namespace tccl {

typedef uint32_t u32x4n __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2n __attribute__((ext_vector_type(2)));
typedef float f32x2n __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2n __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2n __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2n __attribute__((ext_vector_type(2)));

constexpr int kHoldRows = 8, kHoldCols = 128;  // a block of the 8-bit layout
constexpr int kMinExponent = -117;             // the smallest step of a block, 2^-9 * 2^-117, is a normal float: q 2^e is exact

struct NormArgs {
  const char *x, *residual;
  char *summed, *out;
  float *mean, *rstd;
  const void *weight, *bias;
  uint8_t *values, *scales;
  int64_t ld_x, ld_residual, ld_summed, ld_out;  // bytes
  int64_t scale_pitch, value_pitch;              // bytes of a column block's scales, of a row block's values
  int rows, cols, items;                         // items: groups of R rows
  int affine_f32;
  float eps, inv_cols;
};

struct NormGradArgs {
  const char *grad, *x, *grad_summed;
  const uint8_t *values, *scales;
  const float *mean, *rstd;
  const void* weight;
  char* dx;
  float* partial;  // [slot][2][cols]; nullptr: the sums over the rows are made by workgroups of their own, or not wanted
  float *dgamma, *dbeta;  // of those workgroups
  int column_wgs, column_lanes;  // how many there are, ahead of the others; an eighth of their columns
  int64_t ld_grad, ld_x, ld_grad_summed, ld_dx;
  int64_t scale_pitch, value_pitch;
  int rows, cols, items;
  int affine_f32;
  float inv_cols;
};

struct HoldArgs {
  const char* x;
  char* out;
  uint8_t *values, *scales;
  int64_t ld;
  int64_t scale_pitch, value_pitch;
  int rows, cols;
};

#if defined(__HIPCC__)

TCCL_D void renew_words(u32x4n& w) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(w));
#endif
}

// The value exists here (and is not computed later from what it is made of, which would have to be kept).
template <typename W>
TCCL_D void renew_word(W& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(v));
#endif
}

// Instructions stay on their side of this: without it the scheduler converts everything that a thread holds to fp32 first, and
// spills.
TCCL_D void step_by_step() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// Everything here lies in global memory.  (The compiler would take an address that went through a scalar register for one of
// any kind, and wait for LDS at each access.)  kOnce: non-temporal accesses.  Where a wavefront's access covers whole lines,
// which rows of 16-bit activations on 128-byte boundaries give, they copy 512 MiB at 6.4 TB/s instead of 5.8 and read two for
// one written at 6.5 instead of 5.7; where each of several accesses takes a part of every line (8-bit patches, fp32 vectors,
// unaligned rows) they cost a quarter to a third (16384 x 4096 to 8 bits 45 -> 58 us, back 30 -> 41).
template <typename V, bool kOnce = false, typename P>
TCCL_D V got(const P* p) {
  typedef const V __attribute__((address_space(1))) Global;
  if (kOnce) return __builtin_nontemporal_load((Global*)p);
  return *(Global*)p;
}
template <typename V, bool kOnce = false, typename P>
TCCL_D void put(P* p, V v) {
  typedef V __attribute__((address_space(1))) Global;
  if (kOnce)
    __builtin_nontemporal_store(v, (Global*)p);
  else
    *(Global*)p = v;
}

// ---- eight neighbouring values of a row, as they lie in memory ---------------------------------
// Rows may start at any address that their type allows: the accesses say so, and the compiler makes the
// same 16-byte instructions of them.
template <typename T>
struct Eight {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  u32x4n w;
  TCCL_D void zero() { w = (u32x4n){0, 0, 0, 0}; }
  // What is computed from the values again after this is computed again, not kept in registers in between.
  TCCL_D void renew() { renew_words(w); }
  template <bool kOnce>
  TCCL_D void load(const T* p) { w = got<Words, kOnce>(p); }
  template <bool kOnce>
  TCCL_D void store(T* p) const { put<Words, kOnce>(p, w); }
  TCCL_D f32x2n pair(int i) const;
  TCCL_D void set(int i, float a, float b);
  TCCL_D void load_some(const T* p, int n) {
    // The last element stands in for those that do not exist, so that the loads need no branches.
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = got<uint16_t>((const uint16_t*)p + (i < n ? i : n - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (2 * i < n ? h[2 * i] : 0u) | (2 * i + 1 < n ? h[2 * i + 1] << 16 : 0u);
  }
  // From the eight values that end with the row's last to the n (under eight) that the columns from here on have, zeros behind them.
  TCCL_D void settle(int n) {
    const int before = n < 8 ? 8 - n : 0;
    u32x4n v = w;
    if (before & 4) v = (u32x4n){v[2], v[3], 0, 0};
    if (before & 2) v = (u32x4n){v[1], v[2], v[3], 0};
    if (before & 1) v = (u32x4n){v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    w = v;
  }
  TCCL_D void store_some(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) put<uint16_t>((uint16_t*)p + i, (uint16_t)(w[i >> 1] >> (16 * (i & 1))));
  }
};
template <>
TCCL_D f32x2n Eight<__bf16>::pair(int i) const {
  return (f32x2n){__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)};
}
template <>
TCCL_D f32x2n Eight<_Float16>::pair(int i) const {
  const f16x2n h = __builtin_bit_cast(f16x2n, (uint32_t)w[i]);
  return (f32x2n){(float)h[0], (float)h[1]};
}
template <>
TCCL_D void Eight<__bf16>::set(int i, float a, float b) {
  w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(((f32x2n){a, b}), bf16x2n));
}
template <>
TCCL_D void Eight<_Float16>::set(int i, float a, float b) {
  w[i] = __builtin_bit_cast(uint32_t, (f16x2n){(_Float16)a, (_Float16)b});
}
template <>
struct Eight<float> {
  typedef float Words __attribute__((ext_vector_type(4), aligned(4)));
  float v[8];
  TCCL_D void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  template <bool kOnce>
  TCCL_D void load(const float* p) {
    const Words a = got<Words, kOnce>(p), b = got<Words, kOnce>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  }
  template <bool kOnce>
  TCCL_D void store(float* p) const {
    put<Words, kOnce>(p, (Words){v[0], v[1], v[2], v[3]});
    put<Words, kOnce>(p + 4, (Words){v[4], v[5], v[6], v[7]});
  }
  TCCL_D void renew() {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(v[i]));
#endif
  }
  TCCL_D f32x2n pair(int i) const { return (f32x2n){v[2 * i], v[2 * i + 1]}; }
  TCCL_D void set(int i, float a, float b) { v[2 * i] = a, v[2 * i + 1] = b; }
  TCCL_D void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = got<float>(p + (i < n ? i : n - 1));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.f;
  }
  TCCL_D void settle(int n) {
    const int before = n < 8 ? 8 - n : 0;
#pragma unroll
    for (int b = 4; b; b /= 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = before & b ? (i + b < 8 ? v[i + b < 8 ? i + b : 0] : 0.f) : v[i];
    }
  }
  TCCL_D void store_some(float* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) put<float>(p + i, v[i]);
  }
};

// A thread's place in a row whose start is uniform: scalar base, 32-bit offset.  (The compiler would add the offset to the
// tensors' addresses ahead of the loop and keep two vector registers for each.)
template <typename T, typename Byte>
TCCL_D auto in_row(Byte* row, uint32_t off) {
  typedef typename std::conditional<std::is_const<Byte>::value, const T, T>::type Element;
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+s"(row));
#endif
  return (Element*)(row + off);
}

// What the matrices' rows are: of any length and alignment, whole 16-byte vectors on 16-byte boundaries, or those on lines.
enum RowKind { kAnyRows = 0, kVectorRows = 1, kLineRows = 2 };

// The ends of rows that are no whole vectors.  A thread whose columns are the last ones and fewer than eight loads the eight
// that end with them, and moves them to their places once all its loads are on their way: `from` is where it loads, `tail`
// whether its wavefront has such a thread.  (Loads of single values in a branch of their own are waited for row by row:
// 16384 x 1003 backward 58.7 us, so 39.7.)  Rows of fewer than eight columns (narrow) are loaded value by value.
template <int kRows>
struct RowEnds {
  bool narrow;
  TCCL_D RowEnds(int cols) : narrow(kRows == kAnyRows && cols < 8) {}
  template <typename T>
  TCCL_D uint32_t from(int col, int n) const {
    return (uint32_t)(kRows == kAnyRows && !narrow && n > 0 && n < 8 ? col - (8 - n) : col) * (uint32_t)sizeof(T);
  }
  TCCL_D bool tail(int n) const { return kRows == kAnyRows && !narrow && __ballot(n > 0 && n < 8) != 0; }
};
// n: how many of the eight columns exist (8, or fewer at the end of a row; <= 0: none).  Followed by settle(n) where there is a tail.
template <int kRows, bool kOnce = true, typename T>
TCCL_D void load_n(Eight<T>& e, const T* p, int n, const RowEnds<kRows>& ends) {
  if (kRows == kAnyRows ? n > 0 : n >= 8) {
    if (kRows == kAnyRows && ends.narrow)
      e.load_some(p, n);
    else
      e.template load<kOnce && kRows == kLineRows && sizeof(T) == 2>(p);
  } else {
    e.zero();
  }
}
template <int kRows, typename T>
TCCL_D void store_n(const Eight<T>& e, T* p, int n) {
  if (n >= 8)
    e.template store<kRows == kLineRows && sizeof(T) == 2>(p);
  else if (kRows == kAnyRows)
    e.store_some(p, n);
}

// gamma or beta of eight columns, in the activations' type or in fp32; `missing` where there is none.  They are read by
// every workgroup: kept in the caches.
template <typename T, int kRows>
TCCL_D void load_affine(float (&v)[8], const void* p, int f32, int col, int n, float missing, const RowEnds<kRows>& ends) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = missing;
  } else if (f32) {
    Eight<float> e;
    load_n<kRows, false>(e, in_row<float>((const char*)p, ends.template from<float>(col, n)), n, ends);
    if (ends.tail(n)) e.settle(n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e.v[i];
  } else {
    Eight<T> e;
    load_n<kRows, false>(e, in_row<T>((const char*)p, ends.template from<T>(col, n)), n, ends);
    if (ends.tail(n)) e.settle(n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2n q = e.pair(i);
      v[2 * i] = q[0], v[2 * i + 1] = q[1];
    }
  }
}

// ---- sums over lanes, always in the same order ---------------------------------------------------
template <int kControl, int kRows = 0xf>
TCCL_D float moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, kRows, 0xf, false));
}
// Every lane of a row of 16 gets the row's sum.
TCCL_D float sum16(float v) {
  v += moved<0xB1>(v);   // quad_perm [1,0,3,2]
  v += moved<0x4E>(v);   // quad_perm [2,3,0,1]
  v += moved<0x141>(v);  // row_half_mirror
  v += moved<0x140>(v);  // row_mirror
  return v;
}
// The wavefront's sum, uniform.
TCCL_D float sum64(float v) {
  v = sum16(v);
  v += moved<0x142, 0xa>(v);  // row_bcast15 into rows 1 and 3
  v += moved<0x143, 0xc>(v);  // row_bcast31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
TCCL_D uint32_t max16(uint32_t v) {
  uint32_t o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false), v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false), v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false), v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false), v = v > o ? v : o;
  return v;
}
TCCL_D float lane_value(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }

// ---- 8 rows x 8 columns to 8 bits -----------------------------------------------------------------
template <typename T>
struct Bits16;
template <>
struct Bits16<__bf16> {
  static constexpr uint32_t kInf = 0x7f80;
  static constexpr int kTop = 120;  // the exponent of a block that holds values over 448 * 2^119
  static TCCL_D float value(uint32_t b) { return __uint_as_float(b << 16); }
};
template <>
struct Bits16<_Float16> {
  static constexpr uint32_t kInf = 0x7c00;
  static constexpr int kTop = 8;
  static TCCL_D float value(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
};

// The smallest e with amax <= 448 * 2^e, 448 = 1.75 * 2^8, not under kMinExponent.
TCCL_D int held_exponent(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return e < kMinExponent ? kMinExponent : e;
}

// The patch of one lane; 16 neighbouring lanes hold a block.  rows 0..7 of the patch in p[0..7]; what lies outside the
// tensor is zero.  Writes the lane's 64 bytes and, from the first of the 16 lanes, the scale.
// kTurn: four neighbouring lanes turn their 4 x 4 vectors around first, so that a store has 64 bytes in a row of each four, not 16
// of each lane (16384 x 4096 to 8 bits 38.5 -> 34.4 us; in the norm's kernel, short of registers, 8192 x 4096 57.5 -> 59.7).
template <typename T, bool kTurn>
TCCL_D void hold_patch(const Eight<T> (&p)[8], uint8_t* values, uint8_t* scale, bool live, bool first) {
  u16x2n top = {0, 0};
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2n, (uint32_t)(p[r].w[i] & 0x7fff7fffu)));
  // Magnitudes of either 16-bit type are in the order of their bits.
  uint32_t amax = max16(top[0] > top[1] ? top[0] : top[1]);
  bool all_finite = amax < Bits16<T>::kInf;
  if (!all_finite) {  // rare: the largest of what is finite
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = (p[r].w[i >> 1] >> (16 * (i & 1))) & 0x7fffu;
        m = b < Bits16<T>::kInf && b > m ? b : m;
      }
    amax = max16(m);  // the 16 lanes of a block take this branch together
  }
  const int e = held_exponent(Bits16<T>::value(amax));
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  u32x4n q[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {  // columns 2c, 2c + 1
    int lo[2] = {0, 0}, hi[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // rows 4h .. 4h + 3
      f32x2n v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = p[4 * h + r].pair(c);
      lo[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[0][0] * inv, v[1][0] * inv, lo[h], false);
      lo[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2][0] * inv, v[3][0] * inv, lo[h], true);
      hi[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[0][1] * inv, v[1][1] * inv, hi[h], false);
      hi[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2][1] * inv, v[3][1] * inv, hi[h], true);
    }
    q[c] = (u32x4n){(uint32_t)lo[0], (uint32_t)lo[1], (uint32_t)hi[0], (uint32_t)hi[1]};
    step_by_step();
  }
  if (!all_finite) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (((p[r].w[c >> 1] >> (16 * (c & 1))) & 0x7fffu) >= Bits16<T>::kInf)
          q[c >> 1][2 * (c & 1) + (r >> 2)] |= 0x7fu << (8 * (r & 3));  // NaN, of either sign
  }
  if (e == Bits16<T>::kTop) {  // rare: what rounds up to 256 * 2^e is more than the type's largest value; 240 * 2^e is held
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int b = 0; b < 32; b += 8)
          if (((q[c][k] >> b) & 0x7fu) == 0x78u) q[c][k] -= 1u << b;
  }
  const int lane = (int)(threadIdx.x & 63);
  if (kTurn) {
#pragma unroll
    for (int m = 1; m <= 2; m *= 2)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c & m) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int sent = (int)(lane & m ? q[c][k] : q[c + m][k]);
          const uint32_t came = (uint32_t)(m == 1 ? __builtin_amdgcn_update_dpp(0, sent, 0xB1, 0xf, 0xf, false) : __builtin_amdgcn_update_dpp(0, sent, 0x4E, 0xf, 0xf, false));
          q[c][k] = lane & m ? came : q[c][k], q[c + m][k] = lane & m ? q[c + m][k] : came;
        }
      }
  }
  if (live) {
    uint8_t* to = kTurn ? values - (lane & 3) * 48 : values;
#pragma unroll
    for (int c = 0; c < 4; ++c) put<u32x4n>((u32x4n*)(to + c * (kTurn ? 64 : 16)), q[c]);
    if (first) *scale = (uint8_t)(e + 127);
  }
}

// Four rows of two neighbouring columns, from the four codes of each.
TCCL_D void held_quad(uint32_t left, uint32_t right, float scale, f32x2n (&v)[4]) {
  const f32x2n a = __builtin_amdgcn_cvt_pk_f32_fp8((int)left, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)left, true);
  const f32x2n c = __builtin_amdgcn_cvt_pk_f32_fp8((int)right, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)right, true);
  v[0] = (f32x2n){a[0] * scale, c[0] * scale}, v[1] = (f32x2n){a[1] * scale, c[1] * scale};
  v[2] = (f32x2n){b[0] * scale, d[0] * scale}, v[3] = (f32x2n){b[1] * scale, d[1] * scale};
}

// ---- forward ---------------------------------------------------------------------------------------
// blockDim = (64 W, G): G groups of W wavefronts, each with R rows at a time.  (kHold: 1 or 2 of the 128 registers are in scratch; four
// vectors of fp32 with ends of rows to move: 16.)
template <typename T, int R, int NV, bool kHold, int kRows>
__global__ __launch_bounds__(1024, 4) void layer_norm_kernel(NormArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ f32x2n part[2][16][R];  // (sum, sum of squares around the wavefront's mean) of wavefront w, by turns
  const int lane = (int)(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = (int)(blockDim.x >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.y), groups = (int)blockDim.y;
  const int first_part = group * waves;
  const RowEnds<kRows> ends(a.cols);
  int col[NV], left[NV], wave_n = 0;
  uint32_t off[NV], from[NV];
  bool tail = false;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (int)(j * blockDim.x + threadIdx.x) * 8;
    off[j] = (uint32_t)col[j] * (uint32_t)sizeof(T);
    left[j] = a.cols - col[j];
    from[j] = ends.template from<T>(col[j], left[j]);
    tail |= ends.tail(left[j]);
    const int n = a.cols - (j * waves + wave) * 512;
    wave_n += n < 0 ? 0 : n > 512 ? 512 : n;
  }
  const float inv_wave_n = wave_n ? 1.f / (float)wave_n : 0.f;
  // What lane l has of the joining: wavefront l % 16 of row l / 16.
  int join_n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = a.cols - (j * waves + (lane & 15)) * 512;
    join_n += (lane & 15) >= waves || n < 0 ? 0 : n > 512 ? 512 : n;
  }
  const float inv_join_n = join_n ? 1.f / (float)join_n : 0.f;
  constexpr bool kKeep = NV == 1;  // gamma and beta stay in registers
  float gamma[kKeep ? NV : 1][8], beta[kKeep ? NV : 1][8];
  if (kKeep) {
    load_affine<T, kRows>(gamma[0], a.weight, a.affine_f32, col[0], left[0], 1.f, ends);
    load_affine<T, kRows>(beta[0], a.bias, a.affine_f32, col[0], left[0], 0.f, ends);
  }
  int turn = 0;
  for (int base = (int)blockIdx.x * groups; base < a.items; base += (int)gridDim.x * groups, turn ^= 1) {
    const int row0 = (base + group) * R;
    Eight<T> s[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (row0 + r < a.rows && left[j] > 0)
          load_n<kRows>(s[r][j], in_row<T>(a.x + (int64_t)(row0 + r) * a.ld_x, from[j]), left[j], ends);
        else
          s[r][j].zero();
      }
    if (a.residual) {
      Eight<T> t[R][NV];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (row0 + r < a.rows && left[j] > 0)
            load_n<kRows>(t[r][j], in_row<T>(a.residual + (int64_t)(row0 + r) * a.ld_residual, from[j]), left[j], ends);
          else
            t[r][j].zero();
        }
      if (tail) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < NV; ++j) s[r][j].settle(left[j]), t[r][j].settle(left[j]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2n u = s[r][j].pair(i), v = t[r][j].pair(i);
            s[r][j].set(i, u[0] + v[0], u[1] + v[1]);  // rounded to x's type: the norm is that of the sum that is stored
          }
          if (row0 + r < a.rows && left[j] > 0) store_n<kRows>(s[r][j], in_row<T>(a.summed + (int64_t)(row0 + r) * a.ld_summed, off[j]), left[j]);
        }
    }
    if (tail && !a.residual) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NV; ++j) s[r][j].settle(left[j]);
    }
    float sum[R], m2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const f32x2n p0 = s[r][j].pair(0), p1 = s[r][j].pair(1), p2 = s[r][j].pair(2), p3 = s[r][j].pair(3);
        v += ((p0[0] + p0[1]) + (p1[0] + p1[1])) + ((p2[0] + p2[1]) + (p3[0] + p3[1]));
      }
      sum[r] = sum64(v);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = sum[r] * inv_wave_n;
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float d[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2n p = s[r][j].pair(i);
          d[2 * i] = 2 * i < left[j] ? p[0] - mean : 0.f;
          d[2 * i + 1] = 2 * i + 1 < left[j] ? p[1] - mean : 0.f;
        }
        float u = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) u += d[i] * d[i];
        v += u;
      }
      m2[r] = sum64(v);
    }
    float mean[R], rstd[R];
    if (waves == 1) {
#pragma unroll
      for (int r = 0; r < R; ++r) mean[r] = sum[r] * a.inv_cols, rstd[r] = rsqrtf(m2[r] * a.inv_cols + a.eps);
    } else {
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) part[turn][first_part + wave][r] = (f32x2n){sum[r], m2[r]};
      }
      // One barrier per turn: the other half of `part` is written before the next one, and a wavefront that is
      // past that barrier has read this half.
      __syncthreads();
      const int w = (lane & 15) < waves ? (lane & 15) : 0;
#pragma unroll
      for (int r4 = 0; r4 < R; r4 += 4) {
        const int r = r4 + (lane >> 4);
        f32x2n v = part[turn][first_part + w][r < R ? r : R - 1];
        if ((lane & 15) >= waves) v = (f32x2n){0.f, 0.f};
        const float mu = sum16(v[0]) * a.inv_cols;
        const float d = v[0] * inv_join_n - mu;
        const float all = sum16(v[1] + (float)join_n * (d * d));
        const float inv = rsqrtf(all * a.inv_cols + a.eps);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (r4 + k < R) mean[r4 + k] = lane_value(mu, 16 * k), rstd[r4 + k] = lane_value(inv, 16 * k);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NV; ++j) s[r][j].renew();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < a.rows) a.mean[row0 + r] = mean[r], a.rstd[row0 + r] = rstd[r];
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int m = kKeep ? j : 0;
      if (!kKeep) {
        load_affine<T, kRows>(gamma[m], a.weight, a.affine_f32, col[j], left[j], 1.f, ends);
        load_affine<T, kRows>(beta[m], a.bias, a.affine_f32, col[j], left[j], 0.f, ends);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Eight<T> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2n p = s[r][j].pair(i);
          o.set(i, (p[0] - mean[r]) * rstd[r] * gamma[m][2 * i] + beta[m][2 * i],
                (p[1] - mean[r]) * rstd[r] * gamma[m][2 * i + 1] + beta[m][2 * i + 1]);
        }
        if (row0 + r < a.rows && left[j] > 0) store_n<kRows>(o, in_row<T>(a.out + (int64_t)(row0 + r) * a.ld_out, off[j]), left[j]);
      }
      if (NV > 1) step_by_step();
    }
    if constexpr (kHold) {
      static_assert(!kHold || R == kHoldRows, "a row block at a time");
      const int rb = base + group;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Eight<T> p[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) p[r] = s[r][j];
        const int cb = col[j] / kHoldCols;
        // The columns up to a whole block are written too, as zeros.
        const bool live = row0 < a.rows && (int64_t)col[j] * kHoldRows < a.value_pitch;
        hold_patch<T, false>(p, a.values + rb * a.value_pitch + (int64_t)col[j] * kHoldRows, a.scales + cb * a.scale_pitch + rb, live, (lane & 15) == 0);
      }
    }
  }
#endif
}

// ---- backward --------------------------------------------------------------------------------------
// Few rows: workgroup `wg` sums 8 a.column_lanes columns over all rows, reading grad and s a second time (from the caches) instead
// of waiting for the other workgroups' partial sums in a second launch.  column_lanes (4 or 16) lanes side by side, the others
// below each other.  (Eight rows' loads of s in full at a time instead of four: 1000 x 2048 12.4 -> 14.7 us, fewer wavefronts fit.)
constexpr int kMostColumnLanes = 16;
template <typename T, bool kHeld, int kRows>
TCCL_D void sum_columns(const NormGradArgs& a, int wg, float* joined) {
  constexpr int kStep = kHeld ? kHoldRows : 4, Q = 4;
  const int lanes = a.column_lanes, shift = lanes == 4 ? 2 : 4, width = 8 * lanes;
  const int thread = (int)(threadIdx.y * blockDim.x + threadIdx.x), threads = (int)(blockDim.x * blockDim.y);
  const int lane = thread & 63, wave = thread >> 6, waves = threads >> 6;
  const int col = wg * width + (thread & (lanes - 1)) * 8, left = a.cols - col;
  const RowEnds<kRows> ends(8);  // (the rows have that many)
  const uint32_t off = ends.template from<T>(col, left);
  const bool tail = ends.tail(left);
  float dgamma[8], dbeta[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dgamma[i] = dbeta[i] = 0.f;
  for (int row0 = (thread >> shift) * kStep; row0 < a.rows; row0 += (threads >> shift) * kStep) {
    u32x4n q[4];
    float scale = 0.f;
    if (kHeld) {
      const int rb = row0 / kHoldRows;
      const uint8_t* v = a.values + rb * a.value_pitch + (int64_t)col * kHoldRows;
#pragma unroll
      for (int c = 0; c < 4; ++c) q[c] = left > 0 ? got<u32x4n>((const u32x4n*)v + c) : (u32x4n){0, 0, 0, 0};
      if (left > 0) scale = __uint_as_float((uint32_t)a.scales[(col / kHoldCols) * a.scale_pitch + rb] << 23);
    }
#pragma unroll
    for (int h = 0; h < (kHeld ? 2 : 1); ++h) {
      Eight<T> g[Q], s[kHeld ? 1 : Q];
      float mean[Q], rstd[Q];
#pragma unroll
      for (int e = 0; e < Q; ++e) {
        const int row = row0 + 4 * h + e;
        if (row < a.rows) {
          load_n<kRows, false>(g[e], (const T*)(a.grad + (int64_t)row * a.ld_grad + off), left, ends);
          if (!kHeld) load_n<kRows, false>(s[kHeld ? 0 : e], (const T*)(a.x + (int64_t)row * a.ld_x + off), left, ends);
          mean[e] = a.mean[row], rstd[e] = a.rstd[row];
        } else {
          g[e].zero(), mean[e] = rstd[e] = 0.f;
          if (!kHeld) s[kHeld ? 0 : e].zero();
        }
      }
      if (tail) {
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          g[e].settle(left);
          if (!kHeld) s[kHeld ? 0 : e].settle(left);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x2n v[Q];
        if (kHeld)
          held_quad(q[i][h], q[i][2 + h], scale, v);
        else
#pragma unroll
          for (int e = 0; e < Q; ++e) v[e] = s[kHeld ? 0 : e].pair(i);
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          const f32x2n d = g[e].pair(i);
#pragma unroll
          for (int o = 0; o < 2; ++o) dgamma[2 * i + o] += d[o] * ((v[e][o] - mean[e]) * rstd[e]), dbeta[2 * i + o] += d[o];
        }
      }
    }
  }
#pragma unroll
  for (int m = 4; m < 64; m *= 2)
    if (m >= lanes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) dgamma[i] += __shfl_xor(dgamma[i], m), dbeta[i] += __shfl_xor(dbeta[i], m);
    }
  if (lane < lanes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) joined[wave * 2 * width + lane * 8 + i] = dgamma[i], joined[(wave * 2 + 1) * width + lane * 8 + i] = dbeta[i];
  }
  __syncthreads();
  for (int u = thread; u < 2 * width; u += threads) {
    float t = 0.f;
    for (int w = 0; w < waves; ++w) t += joined[w * 2 * width + u];
    const int c = wg * width + (u & (width - 1));
    float* to = u < width ? a.dgamma : a.dbeta;
    if (c < a.cols && to) to[c] = t;
  }
}

// kHeld: s comes from its 8-bit values, R is a row block or half of one.
// Registers: 16 of a vector's are its column sums, 8 more gamma where it stays.  Forms that need more than they have keep the rest in scratch
// memory, read back in every turn: beyond 16384 columns (four vectors) 123 registers of fp32, 188 with ends of rows to move, 11 and 81 of 16
// bits, 85 and 150 from 8 bits; from 8 bits beyond 8192 columns (two vectors) 3 and 30; with ends to move alone, 18 of 16 bits
// a turn ahead beyond 8192 columns and 6 of eight rows from 8 bits.  (python -m tileccl_amd.csrc.check_spills lists them.)
// kAhead: workgroups of up to 512 threads, 512 threads of a CU, whose 256 registers hold two turns: a turn's operands are on their way
// while the turn before is computed (from 8 bits the turns are the halves of a row block, whose codes come with the first).  bf16
// 4096 x 4096 37.3 -> 33.0 us, 4096 x 16384 119 -> 105, from 8 bits 34.6 -> 29.1 and 1030 x 4096 21.1 -> 14.9; fp32 4096 x 4096
// 63 -> 52.  Whole row blocks a turn ahead are more than the registers (16384 x 4096 from 8 bits 89 -> 128 us, so 87), and so are two rows of
// one fp32 vector instead of a row of two (8192 x 4096 119 -> 128 us, so 104).
template <typename T, int R, int NV, bool kHeld, int kRows, bool kAhead>
__global__ __launch_bounds__(kAhead ? 512 : 1024, kAhead ? 2 : 4) void layer_norm_grad_kernel(NormGradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int Q = R < 4 ? R : 4;          // rows taken together
  constexpr bool kHalves = kHeld && kAhead;  // turns are the halves of a row block, whose codes are loaded with the first
  constexpr bool kTwice = kHeld && NV > 1;  // four rows are more than 128 registers: read again (and some are in scratch all the same)
  constexpr int kQuads = kHeld ? R / 4 : 1;  // rows of codes, four in a word
  constexpr bool kKeep = NV == 1 || kAhead;  // gamma stays in registers (a load of it would be waited for with those of the next turn)
  constexpr int KJ = kTwice ? 1 : NV;
  __shared__ f32x2n part[2][16][R];         // (sum g, sum g xh) of wavefront w, by turns
  constexpr bool kGroups = NV == 1 || (kAhead && sizeof(T) == 4);  // whether there may be several groups: of up to eight wavefronts in all
  __shared__ float merged[kGroups ? NV * 7 * 1024 : 16 * 16 * kMostColumnLanes];  // of the groups of a workgroup, or of sum_columns()
  if (!kAhead && (int)blockIdx.x < a.column_wgs) return sum_columns<T, kHeld, kRows>(a, (int)blockIdx.x, merged);
  const int block = (int)blockIdx.x - a.column_wgs, blocks = (int)gridDim.x - a.column_wgs;
  const int lane = (int)(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = (int)(blockDim.x >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.y), groups = (int)blockDim.y;
  const int first_part = group * waves;
  const RowEnds<kRows> ends(a.cols);
  int col[NV], left[NV];
  uint32_t off[NV], from[NV];
  bool tail = false;
  float gamma[kKeep ? NV : 1][8], dgamma[NV][8], dbeta[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (int)(j * blockDim.x + threadIdx.x) * 8;
    off[j] = (uint32_t)col[j] * (uint32_t)sizeof(T);
    left[j] = a.cols - col[j];
    from[j] = ends.template from<T>(col[j], left[j]);
    tail |= ends.tail(left[j]);
    if (kKeep) load_affine<T, kRows>(gamma[j], a.weight, a.affine_f32, col[j], left[j], 1.f, ends);
#pragma unroll
    for (int i = 0; i < 8; ++i) dgamma[j][i] = dbeta[j][i] = 0.f;
  }
  struct Turn {
    int row0;
    Eight<T> g[R][KJ], s[kHeld ? 1 : R][KJ], o[kAhead ? R : 1][kAhead ? NV : 1];
    uint32_t q[kHeld ? KJ : 1][4][kQuads][2];  // column pair, rows, column
    float scale[KJ], mean, rstd;               // the statistics of row `lane`
  };
  uint32_t codes[4][2][2], next_codes[4][2][2];  // kHalves: of this row block and the next; column pair, half, column
  float codes_scale = 0.f, next_scale = 0.f;
  auto fetch = [&](Turn& t, int j, int k) __attribute__((always_inline)) {  // vectors j into place k
    const int row0 = t.row0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r < a.rows) {
        load_n<kRows>(t.g[r][k], in_row<T>(a.grad + (int64_t)(row0 + r) * a.ld_grad, from[j]), left[j], ends);
        if (!kHeld) load_n<kRows>(t.s[kHeld ? 0 : r][k], in_row<T>(a.x + (int64_t)(row0 + r) * a.ld_x, from[j]), left[j], ends);
      } else {
        t.g[r][k].zero();
        if (!kHeld) t.s[kHeld ? 0 : r][k].zero();
      }
    }
    if (kHeld && !kHalves) {
      const int rb = row0 / kHoldRows, half = R == 4 ? row0 / 4 % 2 : 0;
      const bool live = row0 < a.rows && left[j] > 0;
      const uint8_t* v = in_row<const uint8_t>(a.values + rb * a.value_pitch, (uint32_t)col[j] * kHoldRows);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x4n four = live ? got<u32x4n>((const u32x4n*)v + c) : (u32x4n){0, 0, 0, 0};
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          if (R == 4) {
            t.q[kHeld ? k : 0][c][0][o] = half ? four[2 * o + 1] : four[2 * o];
          } else {
#pragma unroll
            for (int h = 0; h < kQuads; ++h) t.q[kHeld ? k : 0][c][h][o] = four[2 * o + h];
          }
        }
      }
      t.scale[k] = live ? __uint_as_float((uint32_t)a.scales[(col[j] / kHoldCols) * a.scale_pitch + rb] << 23) : 0.f;
    }
  };
  auto begin = [&](Turn& t, int base, int half) __attribute__((always_inline)) {
    t.row0 = kHalves ? (base + group) * kHoldRows + 4 * half : (base + group) * R;
    if (kHalves && half == 0) {
      const int rb = base + group;
      const bool live = rb * kHoldRows < a.rows && left[0] > 0;
      const uint8_t* v = in_row<const uint8_t>(a.values + rb * a.value_pitch, (uint32_t)col[0] * kHoldRows);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x4n four = live ? got<u32x4n>((const u32x4n*)v + c) : (u32x4n){0, 0, 0, 0};
#pragma unroll
        for (int o = 0; o < 2; ++o) next_codes[c][0][o] = four[2 * o], next_codes[c][1][o] = four[2 * o + 1];
      }
      next_scale = live ? __uint_as_float((uint32_t)a.scales[(col[0] / kHoldCols) * a.scale_pitch + rb] << 23) : 0.f;
    }
    if (!kTwice) {
#pragma unroll
      for (int j = 0; j < NV; ++j) fetch(t, j, j);
    }
    if (kAhead && a.grad_summed) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (t.row0 + r < a.rows)
            load_n<kRows>(t.o[kAhead ? r : 0][kAhead ? j : 0], in_row<T>(a.grad_summed + (int64_t)(t.row0 + r) * a.ld_grad_summed, from[j]), left[j], ends);
    }
    const bool live = lane < R && t.row0 + lane < a.rows;
    t.mean = live ? a.mean[t.row0 + lane] : 0.f, t.rstd = live ? a.rstd[t.row0 + lane] : 0.f;
  };
  int turn = 0;
  auto finish = [&](Turn& t, int half) __attribute__((always_inline)) {
    const int row0 = t.row0;
    if (kHalves && half == 0) {
      codes_scale = next_scale;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) codes[c][h][0] = next_codes[c][h][0], codes[c][h][1] = next_codes[c][h][1];
    }
    auto settle = [&](int j, int k) __attribute__((always_inline)) {
      if (tail) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          t.g[r][k].settle(left[j]);
          if (!kHeld) t.s[kHeld ? 0 : r][k].settle(left[j]);
        }
      }
    };
    auto values = [&](int k, int i, int h, f32x2n(&v)[4]) __attribute__((always_inline)) {  // s of columns 2i, 2i + 1, rows h Q ..
      if (kHalves)
        held_quad(codes[i][half][0], codes[i][half][1], codes_scale, v);
      else if (kHeld)
        held_quad(t.q[kHeld ? k : 0][i][kHeld ? h : 0][0], t.q[kHeld ? k : 0][i][kHeld ? h : 0][1], t.scale[k], v);
      else
#pragma unroll
        for (int e = 0; e < Q; ++e) v[e] = t.s[kHeld ? 0 : h * Q + e][k].pair(i);
    };
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = lane_value(t.mean, r), rstd[r] = lane_value(t.rstd, r);
    if (!kTwice) {
#pragma unroll
      for (int j = 0; j < NV; ++j) settle(j, j);
    }
    float c1[R], c2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) c1[r] = c2[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = kTwice ? 0 : j, m = kKeep ? j : 0;
      if (kTwice) fetch(t, j, 0), settle(j, 0);
      if (!kKeep) load_affine<T, kRows>(gamma[m], a.weight, a.affine_f32, col[j], left[j], 1.f, ends);
#pragma unroll
      for (int h = 0; h < R / Q; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2n v[4];
          values(k, i, h, v);
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const int r = h * Q + e;
            const f32x2n d = t.g[r][k].pair(i);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float xh = (v[e][o] - mean[r]) * rstd[r];
              const float gd = d[o] * gamma[m][2 * i + o];  // 0 in columns that do not exist
              c1[r] += gd;
              c2[r] += gd * xh;
              dgamma[j][2 * i + o] += d[o] * xh;
              dbeta[j][2 * i + o] += d[o];
            }
          }
#pragma unroll
          for (int o = 0; o < 2; ++o) renew_word(dgamma[j][2 * i + o]), renew_word(dbeta[j][2 * i + o]);
#pragma unroll
          for (int e = 0; e < Q; ++e) renew_word(c1[h * Q + e]), renew_word(c2[h * Q + e]);
          step_by_step();
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) c1[r] = sum64(c1[r]), c2[r] = sum64(c2[r]);
    if (waves > 1) {
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) part[turn][first_part + wave][r] = (f32x2n){c1[r], c2[r]};
      }
      __syncthreads();  // one per turn: see layer_norm_kernel
      const int w = (lane & 15) < waves ? (lane & 15) : 0;
#pragma unroll
      for (int r4 = 0; r4 < R; r4 += 4) {
        const int r = r4 + (lane >> 4);
        f32x2n v = part[turn][first_part + w][r < R ? r : R - 1];
        if ((lane & 15) >= waves) v = (f32x2n){0.f, 0.f};
        const float u = sum16(v[0]), x = sum16(v[1]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (r4 + k < R) c1[r4 + k] = lane_value(u, 16 * k), c2[r4 + k] = lane_value(x, 16 * k);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) c1[r] *= a.inv_cols, c2[r] *= a.inv_cols;
    if (!kTwice) {
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          t.g[r][j].renew();
          if (!kHeld) t.s[kHeld ? 0 : r][j].renew();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int h = 0; h < kQuads; ++h)
            if (kHalves)
              renew_word(codes[c][half][0]), renew_word(codes[c][half][1]);
            else if (kHeld)
              renew_word(t.q[kHeld ? j : 0][c][h][0]), renew_word(t.q[kHeld ? j : 0][c][h][1]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int k = kTwice ? 0 : j, m = kKeep ? j : 0;
      if (kTwice) fetch(t, j, 0), settle(j, 0);
      if (!kKeep) load_affine<T, kRows>(gamma[m], a.weight, a.affine_f32, col[j], left[j], 1.f, ends);
#pragma unroll
      for (int h = 0; h < R / Q; ++h) {
        Eight<T> o[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          const int r = h * Q + e;
          if (!a.grad_summed || row0 + r >= a.rows)
            o[e].zero();
          else if (kAhead)
            o[e] = t.o[kAhead ? r : 0][kAhead ? j : 0];
          else
            load_n<kRows>(o[e], in_row<T>(a.grad_summed + (int64_t)(row0 + r) * a.ld_grad_summed, from[j]), left[j], ends);
        }
        if (tail && a.grad_summed) {
#pragma unroll
          for (int e = 0; e < Q; ++e) o[e].settle(left[j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2n v[4];
          values(k, i, h, v);
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const int r = h * Q + e;
            const f32x2n d = t.g[r][k].pair(i), more = o[e].pair(i);
            float dx[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float xh = (v[e][u] - mean[r]) * rstd[r];
              dx[u] = rstd[r] * (d[u] * gamma[m][2 * i + u] - c1[r] - xh * c2[r]) + more[u];
            }
            o[e].set(i, dx[0], dx[1]);
          }
          step_by_step();
        }
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          const int r = h * Q + e;
          if (row0 + r < a.rows && left[j] > 0) store_n<kRows>(o[e], in_row<T>(a.dx + (int64_t)(row0 + r) * a.ld_dx, off[j]), left[j]);
        }
      }
    }
    turn ^= 1;
  };
  const int step = blocks * groups;
  if constexpr (kHalves) {
    Turn even, odd;
    int base = block * groups;
    bool more = base < a.items;
    if (more) begin(even, base, 0);
    while (more) {
      begin(odd, base, 1);
      step_by_step();
      finish(even, 0);
      base += step;
      more = base < a.items;
      if (more) begin(even, base, 0);
      step_by_step();
      finish(odd, 1);
    }
  } else if constexpr (kAhead) {
    Turn even, odd;
    int base = block * groups;
    bool more = base < a.items;
    if (more) begin(even, base, 0);
    while (more) {
      base += step;
      more = base < a.items;
      if (more) begin(odd, base, 0);
      step_by_step();
      finish(even, 0);
      if (!more) break;
      base += step;
      more = base < a.items;
      if (more) begin(even, base, 0);
      step_by_step();
      finish(odd, 0);
    }
  } else {
    for (int base = block * groups; base < a.items; base += step) {
      Turn t;
      begin(t, base, 0);
      finish(t, 0);
    }
  }
  if (!a.partial) return;
  // The sums of the groups of a workgroup are joined in LDS.
  if constexpr (kGroups) {
    if (groups > 1) {
      const int width = NV * (int)blockDim.x * 8;
      float* mine = merged + (group - 1) * 2 * width;
      if (group > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) mine[col[j] + i] = dgamma[j][i], mine[width + col[j] + i] = dbeta[j][i];
      }
      __syncthreads();
      if (group > 0) return;
      for (int o = 0; o < groups - 1; ++o) {
        const float* other = merged + o * 2 * width;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) dgamma[j][i] += other[col[j] + i], dbeta[j][i] += other[width + col[j] + i];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (left[j] > 0) {
      float* to = a.partial + (int64_t)block * 2 * a.cols + col[j];
      Eight<float> e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = dgamma[j][i];
      store_n<kAnyRows>(e, to, left[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = dbeta[j][i];
      store_n<kAnyRows>(e, to + a.cols, left[j]);
    }
#endif
}

// out[c] = sum over slots of partial[slot][c]; columns [0, cols) go to dgamma, the rest to dbeta.  64 columns per
// workgroup, its wavefronts take every 16th slot.
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, float* dgamma, float* dbeta, int slots, int cols) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ float part[16][64];
  const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
  const int64_t width = 2 * (int64_t)cols, c = (int64_t)blockIdx.x * 64 + lane;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < width) {
    int s = wave;
    for (; s + 48 < slots; s += 64)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += partial[(s + 16 * k) * width + c];
    for (; s < slots; s += 16) v[0] += partial[s * width + c];
  }
  part[wave][lane] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (wave == 0 && c < width) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += part[w][lane];
    if (c < cols) {
      if (dgamma) dgamma[c] = t;
    } else if (dbeta) {
      dbeta[c - cols] = t;
    }
  }
#endif
}

// ---- to 8 bits and back ------------------------------------------------------------------------------
// 256 threads: a patch of 8 rows x 8 columns each; blockIdx.x over 2048 columns, blockIdx.y over row blocks.
template <typename T, int kRows>
__global__ __launch_bounds__(256) void hold_kernel(HoldArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int col = (int)(blockIdx.x * 256 + threadIdx.x) * 8, left = a.cols - col;
  const RowEnds<kRows> ends(a.cols);
  const uint32_t off = ends.template from<T>(col, left);
  const bool tail = ends.tail(left);
  const int row_blocks = (a.rows + kHoldRows - 1) / kHoldRows;
  for (int rb = (int)blockIdx.y; rb < row_blocks; rb += (int)gridDim.y) {
    Eight<T> p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = rb * kHoldRows + r;
      if (row < a.rows && left > 0)
        load_n<kRows>(p[r], in_row<T>(a.x + (int64_t)row * a.ld, off), left, ends);
      else
        p[r].zero();
    }
    if (tail) {
#pragma unroll
      for (int r = 0; r < 8; ++r) p[r].settle(left);
    }
    const bool live = (int64_t)col * kHoldRows < a.value_pitch;
    hold_patch<T, true>(p, a.values + rb * a.value_pitch + (int64_t)col * kHoldRows, a.scales + (col / kHoldCols) * a.scale_pitch + rb, live,
                  (threadIdx.x & 15) == 0);
  }
#endif
}

template <typename T, int kRows>
__global__ __launch_bounds__(256) void restore_kernel(HoldArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int col = (int)(blockIdx.x * 256 + threadIdx.x) * 8, left = a.cols - col;
  const uint32_t off = (uint32_t)col * (uint32_t)sizeof(T);
  const int row_blocks = (a.rows + kHoldRows - 1) / kHoldRows;
  if (left <= 0) return;
  for (int rb = (int)blockIdx.y; rb < row_blocks; rb += (int)gridDim.y) {
    const uint8_t* v = a.values + rb * a.value_pitch + (int64_t)col * kHoldRows;
    u32x4n q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = got<u32x4n>((const u32x4n*)v + c);
    const float scale = __uint_as_float((uint32_t)a.scales[(col / kHoldCols) * a.scale_pitch + rb] << 23);
    Eight<T> o[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        f32x2n x[4];
        held_quad(q[c][h], q[c][2 + h], scale, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[4 * h + k].set(c, x[k][0], x[k][1]);
      }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = rb * kHoldRows + r;
      if (row < a.rows) store_n<kRows>(o[r], in_row<T>(a.out + (int64_t)row * a.ld, off), left);
    }
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
