// AdamW over many tensors: argument checks, launches and the entry points.
#include <hip/hip_runtime.h>

#include <cmath>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_adamw.h"
#include "tccl_host.h"

namespace {

using namespace tccl;

template <typename P, typename G>
void launch(const AdamArgs& a, bool master, bool held, unsigned chunks, hipStream_t stream) {
  const dim3 grid(chunks), threads(held ? kAdamThreadsHeld : kAdamThreads);
  if constexpr (sizeof(P) == 2) {
    if (master) {
      if (held)
        hipLaunchKernelGGL((adamw_kernel<P, G, true, true>), grid, threads, 0, stream, a);
      else
        hipLaunchKernelGGL((adamw_kernel<P, G, true, false>), grid, threads, 0, stream, a);
      return;
    }
  }
  if (held)
    hipLaunchKernelGGL((adamw_kernel<P, G, false, true>), grid, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((adamw_kernel<P, G, false, false>), grid, threads, 0, stream, a);
}

int check(const char* what, const tccl_adamw_desc* d) {
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  if (d->tensors < 0 || (d->tensors && (!d->params || !d->grads || !d->sizes)))
    return reportf(TCCL_ERR_INVALID, "%s: %d tensors, and params, grads and sizes must be non-NULL", what, d->tensors);
  const int p = d->dtype, g = d->grad_dtype;
  if (!((p == TCCL_F32 || p == TCCL_F16 || p == TCCL_BF16) && (g == p || g == TCCL_F32)))
    return reportf(TCCL_ERR_UNSUPPORTED, "%s: params are F32, F16 or BF16, grads of that type or F32", what);
  if (d->master && p == TCCL_F32) return reportf(TCCL_ERR_INVALID, "%s: a master copy of F32 params", what);
  if (d->bits != 8 && d->bits != 32) return reportf(TCCL_ERR_INVALID, "%s: moments of %d bits, must be 8 or 32", what, d->bits);
  if (d->tensors && (!d->first || !d->second || (d->bits == 8 && (!d->first_scales || !d->second_scales))))
    return reportf(TCCL_ERR_INVALID, "%s: moments (and the scales of those in 8 bits) must be non-NULL", what);
  if (((uintptr_t)d->first | (uintptr_t)d->second | (uintptr_t)d->master) & 15) return reportf(TCCL_ERR_UNSUPPORTED, "%s: moments and master must lie on 16 bytes", what);
  if (((uintptr_t)d->step_at | (uintptr_t)d->lr_at | (uintptr_t)d->grad_scale_at) & 3)
    return reportf(TCCL_ERR_INVALID, "%s: step_at, lr_at or grad_scale_at is not aligned to its type", what);
  if (!(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0)) return reportf(TCCL_ERR_INVALID, "%s: betas must lie in [0, 1), got %g and %g", what, d->beta1, d->beta2);
  if (!(d->eps >= 0.0)) return reportf(TCCL_ERR_INVALID, "%s: eps must not be negative, got %g", what, d->eps);
  if (!d->step_at && d->step < 1) return reportf(TCCL_ERR_INVALID, "%s: steps are counted from 1, got %d", what, d->step);
  int64_t blocks = 0;
  for (int i = 0; i < d->tensors; ++i) {
    if (d->sizes[i] < 0) return reportf(TCCL_ERR_INVALID, "%s: tensor %d has %lld elements", what, i, (long long)d->sizes[i]);
    if (!d->sizes[i]) continue;
    if (!d->params[i] || !d->grads[i]) return reportf(TCCL_ERR_INVALID, "%s: tensor %d or its gradient is NULL", what, i);
    if ((uintptr_t)d->params[i] % (p == TCCL_F32 ? 4 : 2) || (uintptr_t)d->grads[i] % (g == TCCL_F32 ? 4 : 2))
      return reportf(TCCL_ERR_INVALID, "%s: tensor %d or its gradient is not aligned to its type", what, i);
    blocks += (d->sizes[i] + kMomentBlock - 1) / kMomentBlock;
    if (d->sizes[i] > (1ll << 38) || blocks > 0xffffffffll)
      return reportf(TCCL_ERR_UNSUPPORTED, "%s: more than 2^32 - 1 blocks of %d elements, or more than 2^38 elements in tensor %d", what, kMomentBlock, i);
  }
  return 0;
}

}  // namespace

extern "C" {

int tccl_adamw(const tccl_adamw_desc* d, void* stream) {
  const char* what = "adamw";
  int rc = check(what, d);
  if (rc) return rc;
  AdamArgs a = {};
  a.first = (char*)d->first, a.second = (char*)d->second;
  a.first_scales = (uint8_t*)d->first_scales, a.second_scales = (uint8_t*)d->second_scales;
  a.master = (float*)d->master;
  a.step_at = d->step_at, a.lr_at = d->lr_at, a.grad_scale_at = d->grad_scale_at;
  a.log_beta1 = std::log(d->beta1), a.log_beta2 = std::log(d->beta2);  // (of 0: -inf, and 1 - b^t = 1)
  a.beta1 = (float)d->beta1, a.beta2 = (float)d->beta2, a.left1 = (float)(1.0 - d->beta1), a.left2 = (float)(1.0 - d->beta2), a.eps = (float)d->eps, a.decay = (float)d->weight_decay;
  a.lr = (float)d->lr, a.grad_scale = (float)d->grad_scale;
  a.step = (uint32_t)d->step;
  a.rate = (float)(d->lr / -std::expm1(d->step * a.log_beta1));
  a.root = (float)(1.0 / std::sqrt(-std::expm1(d->step * a.log_beta2)));
  a.keep = (float)(1.0 - d->lr * d->weight_decay);
  uint64_t chunks = 0;
  uint32_t block = 0;
  auto send = [&]() -> int {
    if (!a.tensors) return 0;
    const bool held = d->bits == 8, master = d->master != nullptr;
    const hipStream_t st = (hipStream_t)stream;
    const unsigned n = (unsigned)chunks;
    const bool wide = d->grad_dtype == TCCL_F32;
    if (d->dtype == TCCL_F32)
      launch<float, float>(a, false, held, n, st);
    else if (d->dtype == TCCL_BF16)
      wide ? launch<__bf16, float>(a, master, held, n, st) : launch<__bf16, __bf16>(a, master, held, n, st);
    else
      wide ? launch<_Float16, float>(a, master, held, n, st) : launch<_Float16, _Float16>(a, master, held, n, st);
    a.tensors = 0, chunks = 0;
    return launched(what);
  };
  // A launch counts its threads in 32 bits.
  constexpr uint64_t kMostChunks = 1u << 23;
  const int chunk = d->bits == 8 ? kAdamChunkHeld : kAdamChunk;
  for (int i = 0; i < d->tensors; ++i) {
    const uint32_t first_block = block;
    block += (uint32_t)((d->sizes[i] + kMomentBlock - 1) / kMomentBlock);
    for (int64_t done = 0; done < d->sizes[i];) {
      if (a.tensors == kAdamTensors || chunks == kMostChunks) {
        rc = send();
        if (rc) return rc;
      }
      const int64_t room = (int64_t)(kMostChunks - chunks) * chunk, n = d->sizes[i] - done < room ? d->sizes[i] - done : room;
      AdamTensor& t = a.t[a.tensors++];
      t.param = (char*)d->params[i] + done * (d->dtype == TCCL_F32 ? 4 : 2);
      t.grad = (const char*)d->grads[i] + done * (d->grad_dtype == TCCL_F32 ? 4 : 2);
      t.n = n, t.block = first_block + (uint32_t)(done / kMomentBlock), t.first_chunk = (uint32_t)chunks;
      chunks += (uint64_t)((n + chunk - 1) / chunk);
      done += n;
    }
  }
  return send();
}

int tccl_adamw_moments(const tccl_adamw_moments_desc* d, void* stream) {
  const char* what = "adamw_moments";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  if (d->blocks < 0 || d->blocks > 0xffffffffll) return reportf(TCCL_ERR_INVALID, "%s: %lld blocks", what, (long long)d->blocks);
  if (!d->blocks) return 0;
  if (!d->first || !d->second || !d->first_scales || !d->second_scales || !d->to_first || !d->to_second) return reportf(TCCL_ERR_INVALID, "%s: moments, scales and results must be non-NULL", what);
  if (((uintptr_t)d->first | (uintptr_t)d->second | (uintptr_t)d->to_first | (uintptr_t)d->to_second) & 15) return reportf(TCCL_ERR_UNSUPPORTED, "%s: moments and results must lie on 16 bytes", what);
  const MomentArgs a = {(const uint8_t*)d->first, (const uint8_t*)d->second, (const uint8_t*)d->first_scales, (const uint8_t*)d->second_scales, (char*)d->to_first, (char*)d->to_second, d->blocks};
  const int64_t wgs = (d->blocks + 15) / 16;
  hipLaunchKernelGGL(moments_kernel, dim3((unsigned)(wgs < 1 << 23 ? wgs : 1 << 23)), dim3(256), 0, (hipStream_t)stream, a);
  return launched(what);
}

}  // extern "C"
