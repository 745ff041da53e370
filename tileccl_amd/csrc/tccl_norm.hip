// Layer norm, its gradients and activations in 8 bits: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>

#include <initializer_list>

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

struct Rows {
  const void* at;
  int64_t ld;
};
// What the rows of all matrices that are there are.
int rows_of(int cols, int size, std::initializer_list<Rows> matrices) {
  if (cols % 8) return kAnyRows;
  uintptr_t bits = 0;
  for (const Rows& m : matrices)
    if (m.at) bits |= (uintptr_t)m.at | (uintptr_t)(m.ld * size);
  return bits % 16 ? kAnyRows : bits % 128 ? kVectorRows : kLineRows;
}

// Whether two matrices of these sizes have no memory in common (their spans: rows between rows count as common).
bool lie_apart(const void* p, int64_t ld_p, const void* q, int64_t ld_q, int rows, int cols, int size) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  const uintptr_t end_a = a + ((int64_t)(rows - 1) * ld_p + cols) * size, end_b = b + ((int64_t)(rows - 1) * ld_q + cols) * size;
  return end_a <= b || end_b <= a;
}

// How a launch of rows x cols is cut: groups of `waves` wavefronts with R rows and NV vectors each, `groups` of them in
// a workgroup.
struct Shape {
  int waves, groups, R, NV, items, wgs, threads;
  bool ahead = false;  // backward: layer_norm_grad_kernel's kAhead
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

// Forward: two rows of a group where they fill the device that way, workgroups for 1536 threads of a CU.  Measured with
// one, two and four rows and 1024 to 4096 threads, or a workgroup for each group of rows: 8192 x 4096 bf16 24.6 us (25.2 with four rows, 30.1 with
// one, 26.3 with all workgroups at once), with a residual 45.5 (48.8, 48.8, 45.3), 16384 x 1024 24.4 (23.8, 26.2, 24.6).
Shape forward_shape(int rows, int cols, bool held, int cus) {
  if (held) return shape_of(rows, cols, kHoldRows, cus, 1024);
  const Shape two = shape_of(rows, cols, 2, cus, 1536);
  return two.NV == 1 && two.items >= 2 * cus * two.groups ? two : shape_of(rows, cols, 1, cus, 1536);
}

// Whether the sums over the rows are made by workgroups of their own (sum_columns) rather than in a second launch.  They read
// a whole column one after the other: 512 x 512 8.8 -> 7.0 us, 1024 x 1024 8.9 -> 7.2, 1024 x 4096 18.3 -> 17.0; but
// 2048 x 1024 10.1 -> 19.4.
bool columns_apart(int rows) { return rows <= 1024; }

// Backward.  Many rows: workgroups of up to 512 threads, 512 of a CU, whose threads are a turn ahead (kAhead), where two turns of
// four vectors (fp32: two; from 8 bits: a row block's halves of four) are no more than 256 registers.  Otherwise one row, or from 8 bits
// eight as long as there are two groups of them for each CU, else four; workgroups of up to 512 threads whose groups join their
// sums, 1024 threads of a CU at most and four turns each (of eight rows, two) if that leaves every CU one: each workgroup's sums are
// written and read again (8192 x 4096 from 8 bits: 50.4 us with two turns, 58.0 with four).
Shape backward_shape(int rows, int cols, int dtype, bool held, int cus) {
  Shape s;
  const bool f32 = dtype == TCCL_F32;
  if (!columns_apart(rows) && cols <= (held ? 4096 : f32 ? 8192 : 16384)) {
    s.ahead = true;
    s.NV = cols > 8192 ? 4 : cols > 4096 || f32 ? 2 : 1, s.R = held ? kHoldRows : (f32 ? 2 : 4) / s.NV;
    s.waves = (cols + 512 * s.NV - 1) / (512 * s.NV);
    s.items = (int)(((int64_t)rows + s.R - 1) / s.R);
    s.groups = 8 / s.waves;
    while (s.groups > 1 && s.items < cus / 2 * s.groups) s.groups /= 2;
    s.threads = 64 * s.waves * s.groups;
    const int wanted = (s.items + s.groups - 1) / s.groups, most = cus * (512 / s.threads);
    s.wgs = wanted < most ? wanted : most;
    return s;
  }
  s = shape_of(rows, cols, held ? kHoldRows : 1, cus, 1024);
  if (held && (s.NV > 1 || s.items < 2 * cus)) s = shape_of(rows, cols, 4, cus, 1024);
  s.groups = s.waves <= 4 ? 8 / s.waves : 1;
  // (sum_columns is quicker with at least 256 threads: 1003 x 1000 from 8 bits 10.3 us with 128 of them)
  while (s.groups > (columns_apart(rows) ? (3 + s.waves) / s.waves : 1) && s.items < cus / 2 * s.groups) s.groups /= 2;
  s.threads = 64 * s.waves * s.groups;
  const int wanted = (s.items + s.groups - 1) / s.groups, most = cus * (s.threads <= 512 ? 1024 / s.threads : 1);
  const int few = wanted / (held ? 2 : 4);
  s.wgs = columns_apart(rows) ? wanted : few < cus ? cus : few;
  if (s.wgs > most && !columns_apart(rows)) s.wgs = most;
  if (s.wgs > wanted) s.wgs = wanted;
  return s;
}

template <typename T, int R, int NV, bool kHold, int kRows>
void launch_forward(const NormArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 block(64 * s.waves, s.groups);
  hipLaunchKernelGGL((layer_norm_kernel<T, R, NV, kHold, kRows>), dim3(s.wgs), block, 0, stream, a);
}

template <typename T, int kRows>
void forward(const NormArgs& a, const Shape& s, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (kRows != kAnyRows)
      if (a.values) return launch_forward<T, 8, 1, true, kRows>(a, s, stream);
  }
  if (s.R == 2) return launch_forward<T, 2, 1, false, kRows>(a, s, stream);
  if (s.NV == 1) return launch_forward<T, 1, 1, false, kRows>(a, s, stream);
  if (s.NV == 2) return launch_forward<T, 1, 2, false, kRows>(a, s, stream);
  return launch_forward<T, 1, 4, false, kRows>(a, s, stream);
}

template <typename T, int R, int NV, bool kHeld, int kRows, bool kAhead = false>
void launch_backward(const NormGradArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 block(64 * s.waves, s.groups);
  hipLaunchKernelGGL((layer_norm_grad_kernel<T, R, NV, kHeld, kRows, kAhead>), dim3(s.wgs + a.column_wgs), block, 0, stream, a);
}

template <typename T, int kRows>
void backward(const NormGradArgs& a, const Shape& s, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (a.values) {
      if (s.ahead) return launch_backward<T, 4, 1, true, kRows, true>(a, s, stream);
      if (s.R == 8) return launch_backward<T, 8, 1, true, kRows>(a, s, stream);
      if (s.NV == 1) return launch_backward<T, 4, 1, true, kRows>(a, s, stream);
      if (s.NV == 2) return launch_backward<T, 4, 2, true, kRows>(a, s, stream);
      return launch_backward<T, 4, 4, true, kRows>(a, s, stream);
    }
    if (s.ahead && s.NV == 1) return launch_backward<T, 4, 1, false, kRows, true>(a, s, stream);
    if (s.ahead && s.NV == 2) return launch_backward<T, 2, 2, false, kRows, true>(a, s, stream);
    if (s.ahead) return launch_backward<T, 1, 4, false, kRows, true>(a, s, stream);
  } else {
    if (s.ahead) return launch_backward<T, 1, 2, false, kRows, true>(a, s, stream);
  }
  if (s.NV == 1) return launch_backward<T, 1, 1, false, kRows>(a, s, stream);
  if (s.NV == 2) return launch_backward<T, 1, 2, false, kRows>(a, s, stream);
  return launch_backward<T, 1, 4, false, kRows>(a, s, stream);
}

int check_sizes(const char* what, int rows, int cols, int dtype, int most_cols) {
  if (rows < 0 || cols < 1) return reportf(TCCL_ERR_INVALID, "%s: rows must not be negative and cols must be positive (got %d, %d)", what, rows, cols);
  if (rows > TCCL_TRAINING_MAX_ROWS) return reportf(TCCL_ERR_UNSUPPORTED, "%s: rows=%d, at most %d", what, rows, TCCL_TRAINING_MAX_ROWS);
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

}  // namespace

extern "C" {

int tccl_hold(const tccl_held_desc* d, void* stream) {
  TCCL_TRY(check_hold("hold", d));
  if (!d->rows) return 0;
  dim3 grid;
  hold_grid(d, &grid);
  const HoldArgs a = hold_args(d);
  const int kind = rows_of(d->cols, 2, {{d->x, d->ld}});
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((kind == kAnyRows ? hold_kernel<__bf16, kAnyRows> : kind == kVectorRows ? hold_kernel<__bf16, kVectorRows> : hold_kernel<__bf16, kLineRows>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((kind == kAnyRows ? hold_kernel<_Float16, kAnyRows> : kind == kVectorRows ? hold_kernel<_Float16, kVectorRows> : hold_kernel<_Float16, kLineRows>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return launched("hold");
}

int tccl_restore(const tccl_held_desc* d, void* stream) {
  TCCL_TRY(check_hold("restore", d));
  if (!d->rows) return 0;
  dim3 grid;
  hold_grid(d, &grid);
  const HoldArgs a = hold_args(d);
  const int kind = rows_of(d->cols, 2, {{d->x, d->ld}});
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((kind == kAnyRows ? restore_kernel<__bf16, kAnyRows> : kind == kVectorRows ? restore_kernel<__bf16, kVectorRows> : restore_kernel<__bf16, kLineRows>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((kind == kAnyRows ? restore_kernel<_Float16, kAnyRows> : kind == kVectorRows ? restore_kernel<_Float16, kVectorRows> : restore_kernel<_Float16, kLineRows>), grid, dim3(256), 0, (hipStream_t)stream, a);
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
  if (d->out == d->summed) return reportf(TCCL_ERR_INVALID, "%s: out and summed are the same memory", what);
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
  const int kind = rows_of(d->cols, size, {{d->x, d->ld_x}, {d->residual, d->ld_residual}, {d->summed, d->ld_summed}, {d->out, d->ld_out}});
  // Eight rows of more columns than these, or with their ends to move, are more than a workgroup's registers: the 8-bit values are then a
  // launch of their own (16384 x 1003 with a residual 42.0 us in one launch, 36.7 in two; 1000 x 1003 15.7, 10.2).
  const bool apart = d->values && (d->cols > 8192 || kind == kAnyRows);
  a.values = apart ? nullptr : (uint8_t*)d->values, a.scales = apart ? nullptr : (uint8_t*)d->scales;
  const Shape s = forward_shape(d->rows, d->cols, a.values != nullptr, cus);
  a.items = s.items;
  // That launch reads the norm's input: x, ahead of the norm, which may write `out` over it, or `summed`, which the norm makes.
  const tccl_held_desc h = {d->residual ? d->summed : const_cast<void*>(d->x), d->values, d->scales, d->residual ? d->ld_summed : d->ld_x,
                            d->rows, d->cols, d->dtype};
  if (apart && !d->residual) TCCL_TRY(tccl_hold(&h, stream));
#define TCCL_FORWARD(T)                                                            \
  (kind == kAnyRows      ? forward<T, kAnyRows>(a, s, (hipStream_t)stream)         \
   : kind == kVectorRows ? forward<T, kVectorRows>(a, s, (hipStream_t)stream)      \
                         : forward<T, kLineRows>(a, s, (hipStream_t)stream))
  if (d->dtype == TCCL_F32)
    TCCL_FORWARD(float);
  else if (d->dtype == TCCL_BF16)
    TCCL_FORWARD(__bf16);
  else
    TCCL_FORWARD(_Float16);
  TCCL_TRY(launched(what));
  return apart && d->residual ? tccl_hold(&h, stream) : 0;
}

int64_t tccl_layer_norm_grad_workspace(int32_t rows, int32_t cols, int32_t dtype, int32_t held) {
  int cus = 0;
  if (check_sizes("layer_norm_grad", rows, cols, dtype, TCCL_NORM_MAX_COLS) || compute_units(&cus)) return -1;
  const Shape s = backward_shape(rows, cols, dtype, held != 0, cus);
  return (int64_t)s.wgs * 2 * cols * 4;
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
  const Shape s = backward_shape(d->rows, d->cols, d->dtype, d->values != nullptr, cus);
  const int slots = s.wgs;
  const bool sums = d->dweight || d->dbias;
  if (d->rows && (!d->workspace || !on16(d->workspace) || d->workspace_bytes < (int64_t)slots * 2 * d->cols * 4))
    return reportf(TCCL_ERR_INVALID, "%s: the workspace has %lld bytes, %lld on 16 are needed", what, (long long)d->workspace_bytes, (long long)slots * 2 * d->cols * 4);
  const int size = size_of(d->dtype);
  const int kind = rows_of(d->cols, size, {{d->grad, d->ld_grad}, {d->x, d->ld_x}, {d->grad_summed, d->ld_grad_summed}, {d->dx, d->ld_dx}});
  // They read grad and x while dx is written: not where those share memory.
  const bool apart = d->rows && d->cols >= 8 && columns_apart(d->rows) && lie_apart(d->dx, d->ld_dx, d->grad, d->ld_grad, d->rows, d->cols, size) &&
                     (!d->x || lie_apart(d->dx, d->ld_dx, d->x, d->ld_x, d->rows, d->cols, size));
  NormGradArgs a;
  a.grad = (const char*)d->grad, a.x = (const char*)d->x, a.grad_summed = (const char*)d->grad_summed;
  a.values = (const uint8_t*)d->values, a.scales = (const uint8_t*)d->scales;
  a.mean = d->mean, a.rstd = d->rstd, a.weight = d->weight, a.dx = (char*)d->dx, a.partial = apart || !sums ? nullptr : (float*)d->workspace;
  a.dgamma = d->dweight, a.dbeta = d->dbias;
  // As many columns as leave every thread of the workgroup one step of rows (16 x 16384: 13.7 us with 32 of them, 7.1 with 128).
  a.column_lanes = (int64_t)d->rows * kMostColumnLanes <= s.threads * (d->values ? kHoldRows : 4) ? kMostColumnLanes : 4;
  a.column_wgs = apart && sums ? (d->cols + 8 * a.column_lanes - 1) / (8 * a.column_lanes) : 0;
  a.ld_grad = d->ld_grad * size, a.ld_x = d->ld_x * size, a.ld_grad_summed = d->ld_grad_summed * size, a.ld_dx = d->ld_dx * size;
  a.scale_pitch = scale_pitch(d->rows), a.value_pitch = value_pitch(d->cols);
  a.rows = d->rows, a.cols = d->cols, a.items = s.items, a.affine_f32 = d->affine_dtype == TCCL_F32;
  a.inv_cols = 1.f / (float)d->cols;
  if (d->rows) {
#define TCCL_BACKWARD(T)                                                           \
  (kind == kAnyRows      ? backward<T, kAnyRows>(a, s, (hipStream_t)stream)        \
   : kind == kVectorRows ? backward<T, kVectorRows>(a, s, (hipStream_t)stream)     \
                         : backward<T, kLineRows>(a, s, (hipStream_t)stream))
    if (d->dtype == TCCL_F32)
      TCCL_BACKWARD(float);
    else if (d->dtype == TCCL_BF16)
      TCCL_BACKWARD(__bf16);
    else
      TCCL_BACKWARD(_Float16);
    TCCL_TRY(launched(what));
  }
  if (sums && !apart)
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((2 * (int64_t)d->cols + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, a.partial, d->dweight,
                       d->dbias, slots, d->cols);
  return launched(what);
}

}  // extern "C"
