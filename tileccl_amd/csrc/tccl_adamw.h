// AdamW over many tensors at once, for gfx950:
//     g = grad * grad_scale,   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// in fp32, on p or, where there is one, on its copy in fp32 ("master"), which then leaves rounded as p.
//
// The moments lie in flat memory, one tensor behind another from a multiple of kMomentBlock elements on.  In 8 bits a block of
// them shares a scale 2^e, a byte e + 127:
//   m  e4m3, e the smallest whole number, at least -117, with max|m| <= 448 * 2^e
//   v  code c from 1 to 254: (1 + ((c - 1) % 8) / 8) * 2^((c - 1) / 8 - 30) * 2^e, code 0: 0, 255: NaN; e = floor(log2(max v)) in
//      -90 .. 127.  No sign, 31 octaves: an element whose v is far below the block's largest must not become 0, its step
//      m / (sqrt(0) + eps) would be a leap; what is positive has at least code 1.
// Maxima are those of finite values; what is not finite is held as NaN.
//
// Rounding is stochastic, and unbiased: b2 = 0.999 moves v by a thousandth of itself a step where neighbouring codes are 6 to 12 % apart,
// and v held to nearest would stay where it is for ever.  Rounded up with a probability that is the fraction of a step above the
// code below, v follows on average; its spread over the 1 / (1 - b2) steps that it remembers is about 20 %, half of that in
// sqrt(v).  The random numbers are 16 bits of a hash of the element's place and the step's number: the same call gives the same bits.
#pragma once

#include "tccl_gemm.h"

namespace tccl {

constexpr int kMomentBlock = 128;
constexpr int kAdamTensors = 100;   // of a launch: its arguments have to fit 4 KiB
constexpr int kAdamThreads = 256;
constexpr int kAdamChunk = 4096;    // elements of a workgroup

struct AdamTensor {
  char *param;
  const char* grad;
  int64_t n;
  uint32_t block;        // where its moments start, in blocks
  uint32_t first_chunk;  // chunks of the tensors ahead of it in this launch
};
struct AdamArgs {
  char *first, *second;                // moments: fp32 or codes
  uint8_t *first_scales, *second_scales;
  float* master;
  const int32_t* step_at;              // where these are read from (NULL: the values below)
  const float *lr_at, *grad_scale_at;
  double log_beta1, log_beta2;         // natural logarithms
  float beta1, beta2, left1, left2;    // left: 1 - beta
  float eps, decay;
  float lr, grad_scale;
  float rate, root, keep;              // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd, where neither step nor lr is read
  uint32_t step;
  int tensors;
  AdamTensor t[kAdamTensors];
};
static_assert(sizeof(AdamArgs) <= 4000, "kernel arguments");

struct MomentArgs {
  const uint8_t *first, *second, *first_scales, *second_scales;
  char *to_first, *to_second;          // bf16
  int64_t blocks;
};

#if defined(__HIPCC__)

// 32 bits for a place in flat memory and a step.  Constants: the golden ratio and fractional parts of square roots, times 2^32, odd.
TCCL_D uint32_t noise_key(uint32_t step, uint32_t high) { return step * 0x9E3779B9u + high * 0xBB67AE85u; }
TCCL_D uint32_t noise(uint32_t place, uint32_t key) {
  uint32_t h = place ^ key;
  h = (h ^ (h >> 16)) * 0x6A09E667u;
  h = (h ^ (h >> 15)) * 0x3C6EF373u;
  return h ^ (h >> 16);
}

// The largest of 16 neighbouring lanes' values, which hold a block.
TCCL_D float max16(float v) {
  auto turn = [](float x, auto by) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(by)::value, 0xf, 0xf, true));
  };
  v = fmaxf(v, turn(v, std::integral_constant<int, 0x128>{}));  // row_ror: 8, 4, 2, 1
  v = fmaxf(v, turn(v, std::integral_constant<int, 0x124>{}));
  v = fmaxf(v, turn(v, std::integral_constant<int, 0x122>{}));
  return fmaxf(v, turn(v, std::integral_constant<int, 0x121>{}));
}
TCCL_D bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

TCCL_D uint32_t first_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return (uint32_t)(e > 10 ? e : 10);
}
TCCL_D uint32_t second_scale(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);
  return (uint32_t)(e > 37 ? e : 37);
}
// `up`: 20 random bits, added below the last bit that stays.  Below 2^-6 e4m3 has steps of 2^-9: with 2^-6 added the value's
// own bits have them, too.
TCCL_D uint32_t first_code(float m, uint32_t scale, uint32_t up) {
  const float y = fabsf(m) * __uint_as_float((254u - scale) << 23);
  const bool small = y < 0.015625f;
  const uint32_t t = __float_as_uint(small ? y + 0.015625f : y) + up;
  const uint32_t code = (t >> 20) - (small ? 968u : 960u);
  return finite(m) ? code | ((__float_as_uint(m) >> 24) & 0x80u) : 0x7fu;
}
TCCL_D uint32_t second_code(float v, uint32_t scale, uint32_t up) {
  const float y = __builtin_amdgcn_ldexpf(v, 127 - (int)scale);
  int code = (int)((__float_as_uint(y) + up) >> 20) - 775;
  const int last = scale == 254u ? 248 : 254;  // 2 * 2^127 is no fp32
  code = code < 1 ? 1 : code > last ? last : code;
  return !finite(v) ? 255u : v > 0.f ? (uint32_t)code : 0u;
}
TCCL_D float second_value(uint32_t code, float scale) {
  const float y = __uint_as_float((code + 775u) << 20) * scale;
  return code == 0u ? 0.f : code == 255u ? __builtin_nanf("") : y;
}
// Codes 4 w .. + 3 of eight.
TCCL_D void first_values(uint32_t codes, float scale, float* m) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  m[0] = lo[0] * scale, m[1] = lo[1] * scale, m[2] = hi[0] * scale, m[3] = hi[1] * scale;
}

// kN elements from `at` on as fp32, and back; `left` of them exist.  Non-temporal: nothing is looked at again before the next step.
template <typename T, int kN>
struct AdamVector {
  typedef T Anywhere __attribute__((ext_vector_type(kN), aligned(sizeof(T))));
  typedef const Anywhere __attribute__((address_space(1))) From;
  typedef Anywhere __attribute__((address_space(1))) To;
  static TCCL_D void get(const char* base, int64_t at, int left, float (&v)[kN]) {
    if (left >= kN) {
      const Anywhere x = __builtin_nontemporal_load((From*)((const T*)base + at));
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = e < left ? (float)((const T*)base)[at + e] : 0.f;
    }
  }
  static TCCL_D void put(char* base, int64_t at, int left, const float (&v)[kN]) {
    if (left >= kN) {
      Anywhere x;
#pragma unroll
      for (int e = 0; e < kN; ++e) x[e] = to_out<T>(v[e]);
      __builtin_nontemporal_store(x, (To*)((T*)base + at));
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < left) ((T*)base)[at + e] = to_out<T>(v[e]);
    }
  }
};

template <typename P, typename G, bool kMaster, bool kHeld>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  // The tensor that this chunk is of: the last one that starts at or before it.
  const int lane = (int)(threadIdx.x & 63);
  int index = -1;
#pragma unroll
  for (int at = 0; at < kAdamTensors; at += 64) {
    const bool here = at + lane < a.tensors && a.t[at + lane < kAdamTensors ? at + lane : 0].first_chunk <= blockIdx.x;
    index += __builtin_popcountll(__builtin_amdgcn_ballot_w64(here));
  }
  const AdamTensor t = a.t[__builtin_amdgcn_readfirstlane(index)];

  uint32_t step = a.step;
  float rate = a.rate, root = a.root, keep = a.keep;
  if (a.step_at || a.lr_at) {
    const float lr = a.lr_at ? *a.lr_at : a.lr;
    if (a.step_at) step = (uint32_t)*a.step_at;
    // 1 - b^t = -expm1(t ln b), without the cancellation
    rate = lr / -expm1f((float)((double)step * a.log_beta1));
    root = 1.f / sqrtf(-expm1f((float)((double)step * a.log_beta2)));
    keep = 1.f - lr * a.decay;
  }
  const float scale = a.grad_scale_at ? *a.grad_scale_at : a.grad_scale;

  const int64_t begin = (int64_t)(blockIdx.x - t.first_chunk) * kAdamChunk;
  // Moments in 32 bits: 4 elements a lane, so that each access of a wavefront is 1 KiB in a row (8 a lane in two accesses each: 67M elements
  // 726 us, 773 non-temporal), two groups of them on their way at a time.  In 8 bits: 8 a lane, 16 lanes a block.
  constexpr int kN = kHeld ? 8 : 4, kGroups = kHeld ? 1 : 2, kTurn = kAdamThreads * kN;
  for (int64_t first = begin + (int)threadIdx.x * kN; first < begin + kAdamChunk; first += kTurn * kGroups) {
    float p[kGroups][kN], g[kGroups][kN], m[kGroups][kN], v[kGroups][kN];
    int left[kGroups];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int64_t at = first + k * kTurn, place = (int64_t)t.block * kMomentBlock + at;
      left[k] = t.n - at < kN ? (t.n - at > 0 ? (int)(t.n - at) : 0) : kN;
      AdamVector<G, kN>::get(t.grad, at, left[k], g[k]);
      if constexpr (kMaster)
        AdamVector<float, kN>::get((const char*)a.master, place, left[k], p[k]);
      else
        AdamVector<P, kN>::get(t.param, at, left[k], p[k]);
      if constexpr (kHeld) {
#pragma unroll
        for (int e = 0; e < kN; ++e) m[k][e] = v[k][e] = 0.f;
        if (left[k]) {
          // (codes of a whole vector are there: a tensor's moments go on to the end of a block)
          const u32x2 cm = __builtin_nontemporal_load((const u32x2*)(a.first + place)), cv = __builtin_nontemporal_load((const u32x2*)(a.second + place));
          const int64_t block = place / kMomentBlock;
          const float sm = __uint_as_float((uint32_t)a.first_scales[block] << 23), sv = __uint_as_float((uint32_t)a.second_scales[block] << 23);
          first_values(cm[0], sm, m[k]);
          first_values(cm[1], sm, m[k] + 4);
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            v[k][e] = second_value((cv[e >> 2] >> (8 * (e & 3))) & 255u, sv);
            if (e >= left[k]) m[k][e] = v[k][e] = 0.f;
          }
        }
      } else {
        AdamVector<float, kN>::get(a.first, place, left[k], m[k]);
        AdamVector<float, kN>::get(a.second, place, left[k], v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int64_t at = first + k * kTurn, place = (int64_t)t.block * kMomentBlock + at;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float d = g[k][e] * scale;
        m[k][e] = a.beta1 * m[k][e] + a.left1 * d;
        v[k][e] = a.beta2 * v[k][e] + a.left2 * (d * d);
        p[k][e] = p[k][e] * keep - rate * m[k][e] * __builtin_amdgcn_rcpf(sqrtf(v[k][e]) * root + a.eps);
      }
      if constexpr (kMaster) AdamVector<float, kN>::put((char*)a.master, place, left[k], p[k]);
      AdamVector<P, kN>::put(t.param, at, left[k], p[k]);
      if constexpr (!kHeld) {
        AdamVector<float, kN>::put(a.first, place, left[k], m[k]);
        AdamVector<float, kN>::put(a.second, place, left[k], v[k]);
      } else {
        // A block's 16 lanes are here together: those past the end have nothing and take part in the block's maximum.
        float top_m = 0.f, top_v = 0.f;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          if (finite(m[k][e])) top_m = fmaxf(top_m, fabsf(m[k][e]));
          if (finite(v[k][e])) top_v = fmaxf(top_v, v[k][e]);
        }
        const uint32_t sm = first_scale(max16(top_m)), sv = second_scale(max16(top_v));
        if (left[k]) {
          const uint32_t key = noise_key(step, (uint32_t)(place >> 32));
          u32x2 cm = {0, 0}, cv = {0, 0};
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            const uint32_t r = noise((uint32_t)place + e, key);
            cm[e >> 2] |= first_code(m[k][e], sm, (r & 0xffffu) << 4) << (8 * (e & 3));
            cv[e >> 2] |= second_code(v[k][e], sv, (r >> 16) << 4) << (8 * (e & 3));
          }
          if (left[k] >= kN) {
            __builtin_nontemporal_store(cm, (u32x2*)(a.first + place));
            __builtin_nontemporal_store(cv, (u32x2*)(a.second + place));
          } else {
#pragma unroll
            for (int e = 0; e < kN; ++e)
              if (e < left[k]) {
                a.first[place + e] = (char)(cm[e >> 2] >> (8 * (e & 3)));
                a.second[place + e] = (char)(cv[e >> 2] >> (8 * (e & 3)));
              }
          }
          if ((place & (kMomentBlock - 1)) == 0) {
            const int64_t block = place / kMomentBlock;
            a.first_scales[block] = (uint8_t)sm;
            a.second_scales[block] = (uint8_t)sv;
          }
        }
      }
    }
  }
#endif
}

// The values that 8-bit moments stand for, exact in bf16: q * 2^e with 4 significant bits.  16 lanes a block.
__global__ __launch_bounds__(256) void moments_kernel(MomentArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < a.blocks * (kMomentBlock / 8); u += (int64_t)gridDim.x * 256) {
    const int64_t block = u / (kMomentBlock / 8);
    const u32x2 cm = *(const u32x2*)(a.first + 8 * u), cv = *(const u32x2*)(a.second + 8 * u);
    const float sm = __uint_as_float((uint32_t)a.first_scales[block] << 23), sv = __uint_as_float((uint32_t)a.second_scales[block] << 23);
    float m[8], v[8];
    first_values(cm[0], sm, m);
    first_values(cm[1], sm, m + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = second_value((cv[e >> 2] >> (8 * (e & 3))) & 255u, sv);
    AdamVector<__bf16, 8>::put(a.to_first, 8 * u, 8, m);
    AdamVector<__bf16, 8>::put(a.to_second, 8 * u, 8, v);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
