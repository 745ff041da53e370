// Layer norm, its gradients and activations in 8 bits: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_host.h"
#include "tccl_norm.h"

static_assert(tccl::kHoldRows == TCCL_HELD_ROWS && tccl::kHoldCols == TCCL_HELD_COLS, "the kernels and the interface agree");

namespace {

using namespace tccl;

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int size_of(int dtype) { return dtype == TCCL_F32 ? 4 : dtype == TCCL_F16 || dtype == TCCL_BF16 ? 2 : 0; }
int64_t row_blocks(int rows) { return ((int64_t)rows + kHoldRows - 1) / kHoldRows; }
int64_t scale_pitch(int rows) { return (row_blocks(rows) + 15) / 16 * 16; }
int64_t value_pitch(int cols) { return ((int64_t)cols + kHoldCols - 1) / kHoldCols * kHoldCols * kHoldRows; }

// How a launch of rows x cols is cut: groups of `waves` wavefronts with R rows and NV vectors each, `groups` of them in
// a workgroup.
struct Shape {
  int waves, groups, R, NV, items, wgs, threads;
};

Shape shape_of(int rows, int cols, int R, int cus, int per_cu_threads) {
  Shape s;
  s.R = R;
  for (s.NV = 1; (cols + 512 * s.NV - 1) / (512 * s.NV) > 16; s.NV *= 2) {}
  s.waves = (cols + 512 * s.NV - 1) / (512 * s.NV);
  s.groups = s.waves >= 3 ? 1 : 4 / s.waves;
  s.threads = 64 * s.waves * s.groups;
  s.items = (int)(((int64_t)rows + R - 1) / R);
  const int wanted = (s.items + s.groups - 1) / s.groups, most = cus * (per_cu_threads / s.threads > 0 ? per_cu_threads / s.threads : 1);
  s.wgs = wanted < most ? wanted : most;
  return s;
}

// Rows of a group: as many as four, unless the rows do not fill the device that way.
Shape choose(int rows, int cols, int dtype, bool held, int cus, int per_cu_threads) {
  if (held) return shape_of(rows, cols, kHoldRows, cus, per_cu_threads);
  Shape s = shape_of(rows, cols, 1, cus, per_cu_threads);
  const int most = s.NV > 1 ? 1 : dtype == TCCL_F32 ? 2 : 4;
  for (int R = most; R > 1; R /= 2) {
    const Shape t = shape_of(rows, cols, R, cus, per_cu_threads);
    if (t.items >= cus * 2 * t.groups) return t;
  }
  return s;
}

template <typename T, int R, int NV, bool kHold>
void launch_forward(const NormArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 block(64 * s.waves, s.groups);
  if constexpr (NV == 1)
    if (s.threads <= 512) {
      hipLaunchKernelGGL((layer_norm_kernel<T, R, NV, kHold, 512>), dim3(s.wgs), block, 0, stream, a);
      return;
    }
  hipLaunchKernelGGL((layer_norm_kernel<T, R, NV, kHold, 1024>), dim3(s.wgs), block, 0, stream, a);
}

template <typename T>
void forward(const NormArgs& a, const Shape& s, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (a.values) return launch_forward<T, 8, 1, true>(a, s, stream);
    if (s.R == 4) return launch_forward<T, 4, 1, false>(a, s, stream);
  }
  if (s.R == 2) return launch_forward<T, 2, 1, false>(a, s, stream);
  if (s.NV == 1) return launch_forward<T, 1, 1, false>(a, s, stream);
  if (s.NV == 2) return launch_forward<T, 1, 2, false>(a, s, stream);
  return launch_forward<T, 1, 4, false>(a, s, stream);
}

template <typename T, int R, int NV, bool kHeld>
void launch_backward(const NormGradArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 block(64 * s.waves, s.groups);
  if constexpr (NV == 1)
    if (s.threads <= 512) {
      hipLaunchKernelGGL((layer_norm_grad_kernel<T, R, NV, kHeld, 512>), dim3(s.wgs), block, 0, stream, a);
      return;
    }
  hipLaunchKernelGGL((layer_norm_grad_kernel<T, R, NV, kHeld, 1024>), dim3(s.wgs), block, 0, stream, a);
}

template <typename T>
void backward(const NormGradArgs& a, const Shape& s, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (a.values) {
      if (s.NV == 1) return launch_backward<T, 8, 1, true>(a, s, stream);
      if (s.NV == 2) return launch_backward<T, 8, 2, true>(a, s, stream);
      return launch_backward<T, 8, 4, true>(a, s, stream);
    }
    if (s.R == 4) return launch_backward<T, 4, 1, false>(a, s, stream);
  }
  if (s.R == 2) return launch_backward<T, 2, 1, false>(a, s, stream);
  if (s.NV == 1) return launch_backward<T, 1, 1, false>(a, s, stream);
  if (s.NV == 2) return launch_backward<T, 1, 2, false>(a, s, stream);
  return launch_backward<T, 1, 4, false>(a, s, stream);
}

int check_sizes(const char* what, int rows, int cols, int dtype, int most_cols) {
  if (rows < 0 || cols < 1) return reportf(TCCL_ERR_INVALID, "%s: rows must not be negative and cols must be positive (got %d, %d)", what, rows, cols);
  if (cols > most_cols) return reportf(TCCL_ERR_UNSUPPORTED, "%s: cols=%d, at most %d", what, cols, most_cols);
  if (!size_of(dtype)) return reportf(TCCL_ERR_UNSUPPORTED, "%s: dtype %d is not F16, BF16 or F32", what, dtype);
  return 0;
}
int check_pitch(const char* what, const char* name, const void* p, int64_t ld, int rows, int cols, int dtype) {
  if (!p && rows) return reportf(TCCL_ERR_INVALID, "%s: %s is NULL", what, name);
  if (rows > 1 && ld < cols) return reportf(TCCL_ERR_INVALID, "%s: %s has a pitch of %lld elements for %d columns", what, name, (long long)ld, cols);
  if ((uintptr_t)p % size_of(dtype)) return reportf(TCCL_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
  return 0;
}
int check_held(const char* what, const void* values, const void* scales, int dtype) {
  if (!values || !scales) return reportf(TCCL_ERR_INVALID, "%s: values and scales go together", what);
  if (dtype == TCCL_F32) return reportf(TCCL_ERR_UNSUPPORTED, "%s: 8-bit values are held of 16-bit types", what);
  if (!on16(values)) return reportf(TCCL_ERR_UNSUPPORTED, "%s: values must lie on 16 bytes", what);
  return 0;
}
#define TCCL_TRY(call)    \
  do {                    \
    const int rc_ = (call); \
    if (rc_) return rc_;  \
  } while (0)

int hold_grid(const tccl_held_desc* d, dim3* grid) {
  const int64_t rb = row_blocks(d->rows);
  *grid = dim3((unsigned)((value_pitch(d->cols) / kHoldRows + 2047) / 2048), (unsigned)(rb < 32768 ? rb : 32768));
  return 0;
}

HoldArgs hold_args(const tccl_held_desc* d) {
  HoldArgs a;
  a.x = (const char*)d->x, a.out = (char*)d->x;
  a.values = (uint8_t*)d->values, a.scales = (uint8_t*)d->scales;
  a.ld = d->ld * size_of(d->dtype);
  a.scale_pitch = scale_pitch(d->rows), a.value_pitch = value_pitch(d->cols);
  a.rows = d->rows, a.cols = d->cols;
  return a;
}

int check_hold(const char* what, const tccl_held_desc* d) {
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  TCCL_TRY(check_sizes(what, d->rows, d->cols, d->dtype, 1 << 27));
  TCCL_TRY(check_pitch(what, "x", d->x, d->ld, d->rows, d->cols, d->dtype));
  if (d->rows) TCCL_TRY(check_held(what, d->values, d->scales, d->dtype));
  return 0;
}

Shape grad_shape(int rows, int cols, int dtype, bool held, int cus) { return choose(rows, cols, dtype, held, cus, 1024); }

}  // namespace

extern "C" {

int tccl_hold(const tccl_held_desc* d, void* stream) {
  TCCL_TRY(check_hold("hold", d));
  if (!d->rows) return 0;
  dim3 grid;
  hold_grid(d, &grid);
  const HoldArgs a = hold_args(d);
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((hold_kernel<__bf16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((hold_kernel<_Float16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return launched("hold");
}

int tccl_restore(const tccl_held_desc* d, void* stream) {
  TCCL_TRY(check_hold("restore", d));
  if (!d->rows) return 0;
  dim3 grid;
  hold_grid(d, &grid);
  const HoldArgs a = hold_args(d);
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((restore_kernel<__bf16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((restore_kernel<_Float16>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return launched("restore");
}

int tccl_layer_norm(const tccl_norm_desc* d, void* stream) {
  const char* what = "layer_norm";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  TCCL_TRY(check_sizes(what, d->rows, d->cols, d->dtype, TCCL_NORM_MAX_COLS));
  TCCL_TRY(check_pitch(what, "x", d->x, d->ld_x, d->rows, d->cols, d->dtype));
  TCCL_TRY(check_pitch(what, "out", d->out, d->ld_out, d->rows, d->cols, d->dtype));
  if ((d->residual != nullptr) != (d->summed != nullptr)) return reportf(TCCL_ERR_INVALID, "%s: residual and summed go together", what);
  if (d->residual) {
    TCCL_TRY(check_pitch(what, "residual", d->residual, d->ld_residual, d->rows, d->cols, d->dtype));
    TCCL_TRY(check_pitch(what, "summed", d->summed, d->ld_summed, d->rows, d->cols, d->dtype));
  }
  if (d->rows && (!d->mean || !d->rstd)) return reportf(TCCL_ERR_INVALID, "%s: mean and rstd are NULL", what);
  if (d->affine_dtype != d->dtype && d->affine_dtype != TCCL_F32) return reportf(TCCL_ERR_UNSUPPORTED, "%s: weight and bias are of x's type or F32", what);
  if ((uintptr_t)d->weight % size_of(d->affine_dtype) || (uintptr_t)d->bias % size_of(d->affine_dtype))
    return reportf(TCCL_ERR_INVALID, "%s: weight or bias is not aligned to its type", what);
  if (d->values || d->scales) TCCL_TRY(check_held(what, d->values, d->scales, d->dtype));
  if (!d->rows) return 0;
  int cus = 0;
  TCCL_TRY(compute_units(&cus));
  const int size = size_of(d->dtype);
  NormArgs a;
  a.x = (const char*)d->x, a.residual = (const char*)d->residual, a.summed = (char*)d->summed, a.out = (char*)d->out;
  a.mean = d->mean, a.rstd = d->rstd, a.weight = d->weight, a.bias = d->bias;
  a.ld_x = d->ld_x * size, a.ld_residual = d->ld_residual * size, a.ld_summed = d->ld_summed * size, a.ld_out = d->ld_out * size;
  a.scale_pitch = scale_pitch(d->rows), a.value_pitch = value_pitch(d->cols);
  a.rows = d->rows, a.cols = d->cols, a.affine_f32 = d->affine_dtype == TCCL_F32;
  a.eps = d->eps, a.inv_cols = 1.f / (float)d->cols;
  // Eight rows of more columns than these are more than a workgroup's registers: the 8-bit values are then a launch
  // of their own.
  const bool apart = d->values && d->cols > 8192;
  a.values = apart ? nullptr : (uint8_t*)d->values, a.scales = apart ? nullptr : (uint8_t*)d->scales;
  const Shape s = choose(d->rows, d->cols, d->dtype, a.values != nullptr, cus, 2048);
  a.items = s.items;
  if (d->dtype == TCCL_F32)
    forward<float>(a, s, (hipStream_t)stream);
  else if (d->dtype == TCCL_BF16)
    forward<__bf16>(a, s, (hipStream_t)stream);
  else
    forward<_Float16>(a, s, (hipStream_t)stream);
  TCCL_TRY(launched(what));
  if (!apart) return 0;
  const tccl_held_desc h = {d->residual ? d->summed : const_cast<void*>(d->x), d->values, d->scales, d->residual ? d->ld_summed : d->ld_x,
                            d->rows, d->cols, d->dtype};
  return tccl_hold(&h, stream);
}

int64_t tccl_layer_norm_grad_workspace(int32_t rows, int32_t cols, int32_t dtype, int32_t held) {
  int cus = 0;
  if (check_sizes("layer_norm_grad", rows, cols, dtype, TCCL_NORM_MAX_COLS) || compute_units(&cus)) return -1;
  const Shape s = grad_shape(rows, cols, dtype, held != 0, cus);
  return (int64_t)s.wgs * s.groups * 2 * cols * 4;
}

int tccl_layer_norm_grad(const tccl_norm_grad_desc* d, void* stream) {
  const char* what = "layer_norm_grad";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  TCCL_TRY(check_sizes(what, d->rows, d->cols, d->dtype, TCCL_NORM_MAX_COLS));
  TCCL_TRY(check_pitch(what, "grad", d->grad, d->ld_grad, d->rows, d->cols, d->dtype));
  TCCL_TRY(check_pitch(what, "dx", d->dx, d->ld_dx, d->rows, d->cols, d->dtype));
  if (d->rows && (d->x != nullptr) == (d->values != nullptr)) return reportf(TCCL_ERR_INVALID, "%s: the norm's input is given as x or as values", what);
  if (d->x) TCCL_TRY(check_pitch(what, "x", d->x, d->ld_x, d->rows, d->cols, d->dtype));
  if (d->values) TCCL_TRY(check_held(what, d->values, d->scales, d->dtype));
  if (d->grad_summed) TCCL_TRY(check_pitch(what, "grad_summed", d->grad_summed, d->ld_grad_summed, d->rows, d->cols, d->dtype));
  if (d->rows && (!d->mean || !d->rstd)) return reportf(TCCL_ERR_INVALID, "%s: mean and rstd are NULL", what);
  if (d->affine_dtype != d->dtype && d->affine_dtype != TCCL_F32) return reportf(TCCL_ERR_UNSUPPORTED, "%s: weight is of grad's type or F32", what);
  if ((uintptr_t)d->weight % size_of(d->affine_dtype)) return reportf(TCCL_ERR_INVALID, "%s: weight is not aligned to its type", what);
  int cus = 0;
  TCCL_TRY(compute_units(&cus));
  const Shape s = grad_shape(d->rows, d->cols, d->dtype, d->values != nullptr, cus);
  const int slots = s.wgs * s.groups;
  if (d->rows && (!d->workspace || !on16(d->workspace) || d->workspace_bytes < (int64_t)slots * 2 * d->cols * 4))
    return reportf(TCCL_ERR_INVALID, "%s: the workspace has %lld bytes, %lld on 16 are needed", what, (long long)d->workspace_bytes, (long long)slots * 2 * d->cols * 4);
  const int size = size_of(d->dtype);
  NormGradArgs a;
  a.grad = (const char*)d->grad, a.x = (const char*)d->x, a.grad_summed = (const char*)d->grad_summed;
  a.values = (const uint8_t*)d->values, a.scales = (const uint8_t*)d->scales;
  a.mean = d->mean, a.rstd = d->rstd, a.weight = d->weight, a.dx = (char*)d->dx, a.partial = (float*)d->workspace;
  a.ld_grad = d->ld_grad * size, a.ld_x = d->ld_x * size, a.ld_grad_summed = d->ld_grad_summed * size, a.ld_dx = d->ld_dx * size;
  a.scale_pitch = scale_pitch(d->rows), a.value_pitch = value_pitch(d->cols);
  a.rows = d->rows, a.cols = d->cols, a.items = s.items, a.affine_f32 = d->affine_dtype == TCCL_F32;
  a.inv_cols = 1.f / (float)d->cols;
  if (d->rows) {
    if (d->dtype == TCCL_F32)
      backward<float>(a, s, (hipStream_t)stream);
    else if (d->dtype == TCCL_BF16)
      backward<__bf16>(a, s, (hipStream_t)stream);
    else
      backward<_Float16>(a, s, (hipStream_t)stream);
    TCCL_TRY(launched(what));
  }
  if (d->dweight || d->dbias)
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((2 * (int64_t)d->cols + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, a.partial, d->dweight,
                       d->dbias, slots, d->cols);
  return launched(what);
}

}  // extern "C"
