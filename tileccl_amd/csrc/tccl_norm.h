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
// 8 rows x 8 columns of a thread are also the unit of the 8-bit layout: values lie as [row block][column][row in block], so a
// thread's patch is 64 contiguous bytes, two neighbouring rows of a column go into one conversion, and the weight gradient
// finds the 8 consecutive rows that a lane of a matrix instruction takes as 8 contiguous bytes, with no transposition.
// 16 neighbouring lanes hold a block of 128 columns, which is one row of the data-parallel primitives.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

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
  float* partial;  // [slot][2][cols]
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

// ---- eight neighbouring values of a row, as they lie in memory ---------------------------------
// Rows may start at any address that their type allows: the accesses say so, and the compiler makes the
// same 16-byte instructions of them.
template <typename T>
struct Eight {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  u32x4n w;
  TCCL_D void zero() { w = (u32x4n){0, 0, 0, 0}; }
  TCCL_D void load(const T* p) { w = *(const Words*)p; }
  TCCL_D void store(T* p) const { *(Words*)p = w; }
  TCCL_D f32x2n pair(int i) const;
  TCCL_D void set(int i, float a, float b);
  TCCL_D void load_some(const T* p, int n) {
    zero();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i >> 1] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i & 1));
  }
  TCCL_D void store_some(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) ((uint16_t*)p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
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
  TCCL_D void load(const float* p) {
    const Words a = *(const Words*)p, b = *(const Words*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  }
  TCCL_D void store(float* p) const {
    *(Words*)p = (Words){v[0], v[1], v[2], v[3]};
    *(Words*)(p + 4) = (Words){v[4], v[5], v[6], v[7]};
  }
  TCCL_D f32x2n pair(int i) const { return (f32x2n){v[2 * i], v[2 * i + 1]}; }
  TCCL_D void set(int i, float a, float b) { v[2 * i] = a, v[2 * i + 1] = b; }
  TCCL_D void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  TCCL_D void store_some(float* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
};

// n: how many of the eight columns exist (8, or fewer at the end of a row; <= 0: none)
template <typename T>
TCCL_D void load_n(Eight<T>& e, const T* p, int n) {
  if (n >= 8)
    e.load(p);
  else
    e.load_some(p, n);
}
template <typename T>
TCCL_D void store_n(const Eight<T>& e, T* p, int n) {
  if (n >= 8)
    e.store(p);
  else
    e.store_some(p, n);
}

// gamma or beta of eight columns, in the activations' type or in fp32; `missing` where there is none
template <typename T>
TCCL_D void load_affine(float (&v)[8], const void* p, int f32, int col, int n, float missing) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = missing;
  } else if (f32) {
    Eight<float> e;
    load_n(e, (const float*)p + col, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e.v[i];
  } else {
    Eight<T> e;
    load_n(e, (const T*)p + col, n);
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
template <typename T>
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
  if (live) {
#pragma unroll
    for (int c = 0; c < 4; ++c) ((u32x4n*)values)[c] = q[c];
    if (first) *scale = (uint8_t)(e + 127);
  }
}

// Rows 4h .. 4h + 3 of a column pair of a held patch: q[c] as hold_patch() writes it.
TCCL_D void held_quad(const u32x4n& q, int h, float scale, f32x2n (&v)[4]) {
  const f32x2n a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
  const f32x2n c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[2 + h], false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[2 + h], true);
  v[0] = (f32x2n){a[0] * scale, c[0] * scale}, v[1] = (f32x2n){a[1] * scale, c[1] * scale};
  v[2] = (f32x2n){b[0] * scale, d[0] * scale}, v[3] = (f32x2n){b[1] * scale, d[1] * scale};
}

// ---- forward ---------------------------------------------------------------------------------------
// blockDim = (64 W, G): G groups of W wavefronts, each with R rows at a time.
template <typename T, int R, int NV, bool kHold, int kThreads>
__global__ __launch_bounds__(kThreads) void layer_norm_kernel(NormArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ f32x2n part[2][16][R];  // (sum, sum of squares around the wavefront's mean) of wavefront w, by turns
  const int lane = (int)(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = (int)(blockDim.x >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.y), groups = (int)blockDim.y;
  const int first_part = group * waves;
  int col[NV], left[NV], wave_n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (int)(j * blockDim.x + threadIdx.x) * 8;
    left[j] = a.cols - col[j];
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
  float gamma[NV][8], beta[NV][8];
  if (kKeep) {
    load_affine<T>(gamma[0], a.weight, a.affine_f32, col[0], left[0], 1.f);
    load_affine<T>(beta[0], a.bias, a.affine_f32, col[0], left[0], 0.f);
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
          load_n(s[r][j], (const T*)(a.x + (int64_t)(row0 + r) * a.ld_x) + col[j], left[j]);
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
            load_n(t[r][j], (const T*)(a.residual + (int64_t)(row0 + r) * a.ld_residual) + col[j], left[j]);
          else
            t[r][j].zero();
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
          if (row0 + r < a.rows && left[j] > 0) store_n(s[r][j], (T*)(a.summed + (int64_t)(row0 + r) * a.ld_summed) + col[j], left[j]);
        }
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
    if (threadIdx.x == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < a.rows) a.mean[row0 + r] = mean[r], a.rstd[row0 + r] = rstd[r];
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!kKeep) {
        load_affine<T>(gamma[j], a.weight, a.affine_f32, col[j], left[j], 1.f);
        load_affine<T>(beta[j], a.bias, a.affine_f32, col[j], left[j], 0.f);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Eight<T> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2n p = s[r][j].pair(i);
          o.set(i, (p[0] - mean[r]) * rstd[r] * gamma[j][2 * i] + beta[j][2 * i],
                (p[1] - mean[r]) * rstd[r] * gamma[j][2 * i + 1] + beta[j][2 * i + 1]);
        }
        if (row0 + r < a.rows && left[j] > 0) store_n(o, (T*)(a.out + (int64_t)(row0 + r) * a.ld_out) + col[j], left[j]);
      }
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
        hold_patch<T>(p, a.values + rb * a.value_pitch + (int64_t)col[j] * kHoldRows, a.scales + cb * a.scale_pitch + rb, live, (lane & 15) == 0);
      }
    }
  }
#endif
}

// ---- backward --------------------------------------------------------------------------------------
// kHeld: s comes from its 8-bit values (then R == 8).
template <typename T, int R, int NV, bool kHeld, int kThreads>
__global__ __launch_bounds__(kThreads) void layer_norm_grad_kernel(NormGradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int Q = R < 4 ? R : 4;   // rows taken together
  __shared__ f32x2n part[2][16][R];  // (sum g, sum g xh) of wavefront w, by turns
  const int lane = (int)(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = (int)(blockDim.x >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.y), groups = (int)blockDim.y;
  const int first_part = group * waves;
  int col[NV], left[NV];
  float gamma[NV][8], dgamma[NV][8], dbeta[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (int)(j * blockDim.x + threadIdx.x) * 8;
    left[j] = a.cols - col[j];
    load_affine<T>(gamma[j], a.weight, a.affine_f32, col[j], left[j], 1.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) dgamma[j][i] = dbeta[j][i] = 0.f;
  }
  int turn = 0;
  for (int base = (int)blockIdx.x * groups; base < a.items; base += (int)gridDim.x * groups, turn ^= 1) {
    const int row0 = (base + group) * R;
    Eight<T> g[R][NV], s[kHeld ? 1 : R][NV];
    u32x4n q[kHeld ? NV : 1][4];
    float scale[NV], mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (row0 + r < a.rows && left[j] > 0) {
          load_n(g[r][j], (const T*)(a.grad + (int64_t)(row0 + r) * a.ld_grad) + col[j], left[j]);
          if (!kHeld) load_n(s[kHeld ? 0 : r][j], (const T*)(a.x + (int64_t)(row0 + r) * a.ld_x) + col[j], left[j]);
        } else {
          g[r][j].zero();
          if (!kHeld) s[kHeld ? 0 : r][j].zero();
        }
      }
    if (kHeld) {
      const int rb = base + group;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const bool live = row0 < a.rows && left[j] > 0;
        const uint8_t* v = a.values + rb * a.value_pitch + (int64_t)col[j] * kHoldRows;
#pragma unroll
        for (int c = 0; c < 4; ++c) q[j][c] = live ? ((const u32x4n*)v)[c] : (u32x4n){0, 0, 0, 0};
        scale[j] = live ? __uint_as_float((uint32_t)a.scales[(col[j] / kHoldCols) * a.scale_pitch + rb] << 23) : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = row0 + r < a.rows;
      mean[r] = live ? a.mean[row0 + r] : 0.f, rstd[r] = live ? a.rstd[row0 + r] : 0.f;
    }
    float c1[R], c2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) c1[r] = c2[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int h = 0; h < R / Q; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2n v[4];
          if (kHeld)
            held_quad(q[kHeld ? j : 0][i], h, scale[j], v);
          else
#pragma unroll
            for (int k = 0; k < Q; ++k) v[k] = s[kHeld ? 0 : h * Q + k][j].pair(i);
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const int r = h * Q + k;
            const f32x2n d = g[r][j].pair(i);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float xh = (v[k][o] - mean[r]) * rstd[r];
              const float gd = d[o] * gamma[j][2 * i + o];  // 0 in columns that do not exist
              c1[r] += gd;
              c2[r] += gd * xh;
              dgamma[j][2 * i + o] += d[o] * xh;
              dbeta[j][2 * i + o] += d[o];
            }
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
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int h = 0; h < R / Q; ++h) {
        Eight<T> o[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int r = h * Q + k;
          if (a.grad_summed && row0 + r < a.rows && left[j] > 0)
            load_n(o[k], (const T*)(a.grad_summed + (int64_t)(row0 + r) * a.ld_grad_summed) + col[j], left[j]);
          else
            o[k].zero();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2n v[4];
          if (kHeld)
            held_quad(q[kHeld ? j : 0][i], h, scale[j], v);
          else
#pragma unroll
            for (int k = 0; k < Q; ++k) v[k] = s[kHeld ? 0 : h * Q + k][j].pair(i);
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const int r = h * Q + k;
            const f32x2n d = g[r][j].pair(i), more = o[k].pair(i);
            float dx[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float xh = (v[k][e] - mean[r]) * rstd[r];
              dx[e] = rstd[r] * (d[e] * gamma[j][2 * i + e] - c1[r] - xh * c2[r]) + more[e];
            }
            o[k].set(i, dx[0], dx[1]);
          }
        }
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int r = h * Q + k;
          if (row0 + r < a.rows && left[j] > 0) store_n(o[k], (T*)(a.dx + (int64_t)(row0 + r) * a.ld_dx) + col[j], left[j]);
        }
      }
  }
  const int64_t slot = (int64_t)blockIdx.x * groups + group;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (left[j] > 0) {
      float* to = a.partial + slot * 2 * a.cols + col[j];
      Eight<float> e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = dgamma[j][i];
      store_n(e, to, left[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = dbeta[j][i];
      store_n(e, to + a.cols, left[j]);
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
template <typename T>
__global__ __launch_bounds__(256) void hold_kernel(HoldArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int col = (int)(blockIdx.x * 256 + threadIdx.x) * 8, left = a.cols - col;
  const int row_blocks = (a.rows + kHoldRows - 1) / kHoldRows;
  for (int rb = (int)blockIdx.y; rb < row_blocks; rb += (int)gridDim.y) {
    Eight<T> p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = rb * kHoldRows + r;
      if (row < a.rows && left > 0)
        load_n(p[r], (const T*)(a.x + (int64_t)row * a.ld) + col, left);
      else
        p[r].zero();
    }
    const bool live = (int64_t)col * kHoldRows < a.value_pitch;
    hold_patch<T>(p, a.values + rb * a.value_pitch + (int64_t)col * kHoldRows, a.scales + (col / kHoldCols) * a.scale_pitch + rb, live,
                  (threadIdx.x & 15) == 0);
  }
#endif
}

template <typename T>
__global__ __launch_bounds__(256) void restore_kernel(HoldArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int col = (int)(blockIdx.x * 256 + threadIdx.x) * 8, left = a.cols - col;
  const int row_blocks = (a.rows + kHoldRows - 1) / kHoldRows;
  if (left <= 0) return;
  for (int rb = (int)blockIdx.y; rb < row_blocks; rb += (int)gridDim.y) {
    const uint8_t* v = a.values + rb * a.value_pitch + (int64_t)col * kHoldRows;
    u32x4n q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = ((const u32x4n*)v)[c];
    const float scale = __uint_as_float((uint32_t)a.scales[(col / kHoldCols) * a.scale_pitch + rb] << 23);
    Eight<T> o[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        f32x2n x[4];
        held_quad(q[c], h, scale, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[4 * h + k].set(c, x[k][0], x[k][1]);
      }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = rb * kHoldRows + r;
      if (row < a.rows) store_n(o[r], (T*)(a.out + (int64_t)row * a.ld) + col, left);
    }
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
