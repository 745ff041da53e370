// AdamW over many tensors at once, for gfx950:
//     g = grad * grad_scale,   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// in fp32 (under the root a v below 2^-126 counts as 0), on p or, where there is one, on its copy in fp32 ("master"), which then leaves rounded as p.
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
// Threads of a workgroup, and elements of a thread: each has one turn.  Moments in 32 bits: 4 elements, so that each access of a wavefront is 1 KiB in
// a row.  In 8 bits: 8, 16 lanes a block (4, 32 lanes, 585 us).  Larger workgroups and several turns are slower (128M weights in 32 bits 617 us; 256 threads
// 629, 512 648, with two turns 673; 197M in 8 bits 563; 128 threads 572, two turns 575).
constexpr int kAdamThreads = 128, kAdamThreadsHeld = 256;
constexpr int kAdamChunk = 4 * kAdamThreads, kAdamChunkHeld = 8 * kAdamThreadsHeld;

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
TCCL_D uint32_t max16(uint32_t v) {
  auto turn = [](uint32_t x, auto by) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(by)::value, 0xf, 0xf, true); };
  auto most = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
  v = most(v, turn(v, std::integral_constant<int, 0x128>{}));  // row_ror: 8, 4, 2, 1
  v = most(v, turn(v, std::integral_constant<int, 0x124>{}));
  v = most(v, turn(v, std::integral_constant<int, 0x122>{}));
  return most(v, turn(v, std::integral_constant<int, 0x121>{}));
}
// Magnitudes are compared by their bits, among which what is not finite stands above all others.
constexpr uint32_t kNotFinite = 0x7f800000u;
TCCL_D uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

TCCL_D uint32_t first_scale(uint32_t top) {
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
  return (uint32_t)(e > 10 ? e : 10);
}
TCCL_D uint32_t second_scale(uint32_t top) { return top >> 23 > 37u ? top >> 23 : 37u; }
// Byte e of `into` becomes the code of m / 2^e, of finite values.  The conversion adds its random number below the last bit that stays,
// denormal or not; of the 32 bits that it takes the upper 20 count here, and 16 of them are random (4M values and random numbers of every magnitude
// gave the codes of the definition).
template <int kByte>
TCCL_D uint32_t first_code(float m, float inverse, uint32_t random, uint32_t into) {
  return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(m * inverse, (int)(random << 16), (int)into, kByte);
}
TCCL_D uint32_t second_code(float v, uint32_t scale, uint32_t random) {
  const float y = __builtin_amdgcn_ldexpf(v, 127 - (int)scale);
  const int code = (int)((__float_as_uint(y) + ((random >> 12) & 0xffff0u)) >> 20) - 775;
  return v > 0.f ? (uint32_t)(code > 1 ? code : 1) : 0u;
}
// The values of four codes.
TCCL_D void first_values(uint32_t codes, float scale, float* m) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  m[0] = lo[0] * scale, m[1] = lo[1] * scale, m[2] = hi[0] * scale, m[3] = hi[1] * scale;
}
TCCL_D void second_values(uint32_t codes, float scale, float* v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t code = (codes >> (8 * e)) & 255u;
    v[e] = code ? __uint_as_float((code + 775u) << 20) * scale : 0.f;
  }
  if ((~codes - 0x01010101u) & codes & 0x80808080u)  // a byte of ~codes may be 0: one of 255 is NaN
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (((codes >> (8 * e)) & 255u) == 255u) v[e] = __builtin_nanf("");
}

// kN elements from `at` on as fp32, and back; `left` of them exist.  Non-temporal, as nothing is looked at again before the next step, but where a
// wavefront's access has gaps, which the next one fills.
template <typename T, int kN>
struct AdamVector {
  static constexpr bool kGaps = sizeof(T) * kN > 16;
  typedef T Anywhere __attribute__((ext_vector_type(kN), aligned(sizeof(T))));
  typedef const Anywhere __attribute__((address_space(1))) From;
  typedef Anywhere __attribute__((address_space(1))) To;
  static TCCL_D void get(const char* base, int64_t at, int left, float (&v)[kN]) {
    if (left >= kN) {
      const Anywhere x = kGaps ? *(From*)((const T*)base + at) : __builtin_nontemporal_load((From*)((const T*)base + at));
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
      if (kGaps)
        *(To*)((T*)base + at) = x;
      else
        __builtin_nontemporal_store(x, (To*)((T*)base + at));
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < left) ((T*)base)[at + e] = to_out<T>(v[e]);
    }
  }
};

// Bound by memory: bf16 weights with fp32 copy, gradients and moments, 128M of them, 617 us, 6.2 TB/s with as many writes as reads (a
// plain copy of 512 MiB 5.3 to 6.1); moments in 8 bits, 197M with bf16 gradients, 563 us, 5.6 TB/s, the vector units half busy.
template <typename P, typename G, bool kMaster, bool kHeld>
__global__ __launch_bounds__(kHeld ? kAdamThreadsHeld : kAdamThreads) void adamw_kernel(AdamArgs a) {
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

  constexpr int kN = kHeld ? 8 : 4;
  const int64_t at = (int64_t)(blockIdx.x - t.first_chunk) * (kHeld ? kAdamChunkHeld : kAdamChunk) + (int)threadIdx.x * kN, place = (int64_t)t.block * kMomentBlock + at;
  const int left = t.n - at < kN ? (t.n - at > 0 ? (int)(t.n - at) : 0) : kN;
  float p[kN], g[kN], m[kN], v[kN];
  AdamVector<G, kN>::get(t.grad, at, left, g);
  if constexpr (kMaster)
    AdamVector<float, kN>::get((const char*)a.master, place, left, p);
  else
    AdamVector<P, kN>::get(t.param, at, left, p);
  if constexpr (kHeld) {
#pragma unroll
    for (int e = 0; e < kN; ++e) m[e] = v[e] = 0.f;
    if (left) {
      // (codes of a whole vector are there: a tensor's moments go on to the end of a block)
      const u32x2 cm = __builtin_nontemporal_load((const u32x2*)(a.first + place)), cv = __builtin_nontemporal_load((const u32x2*)(a.second + place));
      const int64_t block = place / kMomentBlock;
      const float sm = __uint_as_float((uint32_t)a.first_scales[block] << 23), sv = __uint_as_float((uint32_t)a.second_scales[block] << 23);
      first_values(cm[0], sm, m);
      first_values(cm[1], sm, m + 4);
      second_values(cv[0], sv, v);
      second_values(cv[1], sv, v + 4);
      if (left < kN)
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (e >= left) m[e] = v[e] = 0.f;
    }
  } else {
    AdamVector<float, kN>::get(a.first, place, left, m);
    AdamVector<float, kN>::get(a.second, place, left, v);
  }
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    const float d = g[e] * scale;
    m[e] = a.beta1 * m[e] + a.left1 * d;
    v[e] = a.beta2 * v[e] + a.left2 * (d * d);
    p[e] = p[e] * keep - rate * m[e] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[e]) * root + a.eps);
  }
  if constexpr (kMaster) AdamVector<float, kN>::put((char*)a.master, place, left, p);
  AdamVector<P, kN>::put(t.param, at, left, p);
  if constexpr (!kHeld) {
    AdamVector<float, kN>::put(a.first, place, left, m);
    AdamVector<float, kN>::put(a.second, place, left, v);
  } else {
    // A block's 16 lanes are here together: those past the end have nothing and take part in the block's maximum.
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const uint32_t bm = magnitude(m[e]), bv = magnitude(v[e]);
      top_m = bm > top_m ? bm : top_m, top_v = bv > top_v ? bv : top_v;
    }
    top_m = max16(top_m), top_v = max16(top_v);
    // Blocks with something that is not finite, or with a v that may be rounded up to 2^128.
    const bool odd = top_m >= kNotFinite || top_v >= 254u << 23;
    if (odd) {
      top_m = top_v = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const uint32_t bm = magnitude(m[e]), bv = magnitude(v[e]);
        if (bm < kNotFinite && bm > top_m) top_m = bm;
        if (bv < kNotFinite && bv > top_v) top_v = bv;
      }
      top_m = max16(top_m), top_v = max16(top_v);
    }
    const uint32_t sm = first_scale(top_m), sv = second_scale(top_v);
    if (left) {
      const float inverse = __uint_as_float((254u - sm) << 23);
      const uint32_t key = noise_key(step, (uint32_t)(place >> 32));
      uint32_t random[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) random[e] = noise((uint32_t)place + e, key);
      u32x2 cm, cv;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        cm[w] = first_code<3>(m[4 * w + 3], inverse, random[4 * w + 3],
                              first_code<2>(m[4 * w + 2], inverse, random[4 * w + 2],
                                            first_code<1>(m[4 * w + 1], inverse, random[4 * w + 1], first_code<0>(m[4 * w], inverse, random[4 * w], 0u))));
        cv[w] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) cv[w] |= second_code(v[4 * w + e], sv, random[4 * w + e]) << (8 * e);
      }
      if (odd) {
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const uint32_t shift = 8 * (e & 3), byte = 255u << shift, code = (cv[e >> 2] >> shift) & 255u;
          if (magnitude(m[e]) >= kNotFinite) cm[e >> 2] = (cm[e >> 2] & ~byte) | 0x7fu << shift;
          if (magnitude(v[e]) >= kNotFinite)
            cv[e >> 2] |= byte;
          else if (sv == 254u && code > 248u)  // 2 * 2^127 is no fp32
            cv[e >> 2] = (cv[e >> 2] & ~byte) | 248u << shift;
        }
      }
      if (left >= kN) {
        __builtin_nontemporal_store(cm, (u32x2*)(a.first + place));
        __builtin_nontemporal_store(cv, (u32x2*)(a.second + place));
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (e < left) {
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
#endif
}

// The values that 8-bit moments stand for, exact in bf16: q * 2^e with 4 significant bits.  16 lanes a block.  197M 187 us, 6.3 TB/s (in turns
// of 16384 workgroups 214).
__global__ __launch_bounds__(256) void moments_kernel(MomentArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < a.blocks * (kMomentBlock / 8); u += (int64_t)gridDim.x * 256) {
    const int64_t block = u / (kMomentBlock / 8);
    const u32x2 cm = __builtin_nontemporal_load((const u32x2*)(a.first + 8 * u)), cv = __builtin_nontemporal_load((const u32x2*)(a.second + 8 * u));
    const float sm = __uint_as_float((uint32_t)a.first_scales[block] << 23), sv = __uint_as_float((uint32_t)a.second_scales[block] << 23);
    float m[8], v[8];
    first_values(cm[0], sm, m);
    first_values(cm[1], sm, m + 4);
    second_values(cv[0], sv, v);
    second_values(cv[1], sv, v + 4);
    AdamVector<__bf16, 8>::put(a.to_first, 8 * u, 8, m);
    AdamVector<__bf16, 8>::put(a.to_second, 8 * u, 8, v);
  }
#endif
}

#endif  // __HIPCC__

}  // namespace tccl
