// Weight gradients from activations in 8 bits: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>
#include <initializer_list>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_host.h"
#include "tccl_weight.h"

namespace {

using namespace tccl;

// The kernels: 256 x 256 tiles; 128 x 128 by eight wavefronts (two groups); 128 x 128 by four, two workgroups per CU.
enum Kind { kLarge, kPairs, kSmall };

struct Cut {
  Kind kind;
  int tiles_h, tiles_n, steps, splits, steps_per_split;
};

Cut cut_of(Kind kind, int splits, int rows, int cols, int outputs) {
  const int edge = kind == kLarge ? 256 : 128;
  Cut c;
  c.kind = kind;
  c.tiles_h = (cols + edge - 1) / edge, c.tiles_n = (outputs + edge - 1) / edge;
  c.steps = (rows + 63) / 64;
  c.steps_per_split = (c.steps + splits - 1) / splits;
  c.splits = c.steps ? (c.steps + c.steps_per_split - 1) / c.steps_per_split : 1;
  return c;
}

// An estimate of a launch's microseconds, fitted to shapes of 64 to 16384 tokens and 64 to 7168 inputs and outputs with every kind and up
// to 128 splits.  Of the thirty it was then checked at, what it chose took at most 7 % longer than the best (9000 x 130 x 3000: 28.2, best
// 26.4 us).  A step of 64 tokens: 1.53 us of a 256 tile (less where CUs are idle: the clock is higher), 1.0 of two steps by two groups,
// 0.95 of two workgroups on a CU, 0.65 of one alone there; what is left over behind full rounds fills gaps of theirs, 0.45.
double estimate(const Cut& c, int cols, int outputs, int cus) {
  const int64_t wgs = (int64_t)c.tiles_h * c.tiles_n * c.splits, steps = c.steps_per_split;
  const double out_mb = 4e-6 * cols * outputs;
  double us = 5.0 + out_mb / 5.0;
  if (c.kind == kLarge)
    us += (wgs + cus - 1) / cus * (wgs < cus ? 1.2 + 0.33 * wgs / cus : 1.53) * steps;
  else if (c.kind == kPairs)
    us += 1.0 + (wgs + cus - 1) / cus * ((steps + 1) / 2);
  else
    us += wgs / (2 * cus) * 0.95 * steps + (wgs % (2 * cus) > cus ? 0.95 : wgs % (2 * cus) == 0 ? 0.0 : wgs > 2 * cus ? 0.45 : 0.65) * steps;
  if (c.splits > 1) us += 3.5 + 2.0 * c.splits * out_mb / 5.0;  // the partial sums there and back, and a second launch
  return us;
}

Cut choose(int rows, int cols, int outputs, int cus) {
  Cut best = cut_of(kSmall, 1, rows, cols, outputs);
  double least = estimate(best, cols, outputs, cus);
  for (const Kind kind : {kLarge, kPairs, kSmall})
    for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (splits > 1 && (rows + 63) / 64 < 2 * splits) break;
      const Cut c = cut_of(kind, splits, rows, cols, outputs);
      const double us = estimate(c, cols, outputs, cus);
      if (us < least) best = c, least = us;
    }
  return best;
}

int64_t partial_pitch(int cols) { return ((int64_t)cols + 3) / 4 * 4; }
int64_t partial_rows(int rows, int cols) { return (int64_t)rows * partial_pitch(cols); }

template <typename T, typename OutT, bool kTransposed>
int launch(const WeightArgs& a, const Cut& c, hipStream_t stream) {
  const dim3 wgs((unsigned)(a.xcds * a.per_xcd));
  if (c.kind == kLarge)
    hipLaunchKernelGGL((weight_gradient_kernel<T, OutT, 256, 256, kTransposed, 1>), wgs, dim3(512), 0, stream, a);
  else if (c.kind == kPairs)
    hipLaunchKernelGGL((weight_gradient_kernel<T, OutT, 128, 128, kTransposed, 2>), wgs, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((weight_gradient_kernel<T, OutT, 128, 128, kTransposed, 1>), wgs, dim3(256), 0, stream, a);
  return launched("weight_gradient");
}

template <typename T, typename OutT>
int launch_out(const WeightArgs& a, const Cut& c, bool transposed, hipStream_t stream) {
  const int rc = transposed ? launch<T, OutT, true>(a, c, stream) : launch<T, OutT, false>(a, c, stream);
  if (rc || c.splits == 1) return rc;
  WeightSumArgs s;
  s.rows = transposed ? a.outputs : a.cols, s.cols = transposed ? a.cols : a.outputs;
  s.partial = a.partial, s.add = a.add, s.out = a.out;
  s.ld_partial = a.ld_partial, s.ld_add = a.ld_add, s.ld_out = a.ld_out, s.slice = s.rows * a.ld_partial;
  s.splits = c.splits;
  const int64_t units = (int64_t)s.rows * ((s.cols + 3) / 4);
  const int64_t wgs = (units + 255) / 256;
  hipLaunchKernelGGL((weight_sum_kernel<OutT>), dim3((unsigned)(wgs < 4096 ? wgs : 4096)), dim3(256), 0, stream, s);
  return launched("weight_gradient");
}

int check_sizes(const char* what, int rows, int cols, int outputs) {
  if (rows < 0 || cols < 1 || outputs < 1)
    return reportf(TCCL_ERR_INVALID, "%s: rows must not be negative, cols and outputs must be positive (got %d, %d, %d)", what, rows, cols, outputs);
  if (rows > TCCL_TRAINING_MAX_ROWS) return reportf(TCCL_ERR_UNSUPPORTED, "%s: rows=%d, at most %d", what, rows, TCCL_TRAINING_MAX_ROWS);
  if (cols > 1 << 24 || outputs > 1 << 24) return reportf(TCCL_ERR_UNSUPPORTED, "%s: %d x %d outputs, at most %d of either", what, cols, outputs, 1 << 24);
  return 0;
}

int size_of(int dtype) { return dtype == TCCL_F32 ? 4 : dtype == TCCL_F16 || dtype == TCCL_BF16 ? 2 : 0; }

}  // namespace

extern "C" {

int64_t tccl_weight_gradient_workspace(int32_t rows, int32_t cols, int32_t outputs) {
  int cus = 0;
  if (check_sizes("weight_gradient", rows, cols, outputs) || compute_units(&cus)) return -1;
  const Cut c = choose(rows, cols, outputs, cus);
  if (c.splits == 1) return 0;
  const int64_t kn = partial_rows(cols, outputs), nk = partial_rows(outputs, cols);
  return 4 * c.splits * (kn > nk ? kn : nk);
}

int tccl_weight_gradient_cut(int32_t rows, int32_t cols, int32_t outputs, int32_t compute_units, int32_t* edge, int32_t* groups, int32_t* splits,
                             int32_t* steps_per_split) {
  const int rc = check_sizes("weight_gradient_cut", rows, cols, outputs);
  if (rc) return rc;
  if (compute_units < 1 || !edge || !groups || !splits || !steps_per_split)
    return reportf(TCCL_ERR_INVALID, "weight_gradient_cut: %d compute units, or a NULL result", compute_units);
  const Cut c = choose(rows, cols, outputs, compute_units);
  *edge = c.kind == kLarge ? 256 : 128, *groups = c.kind == kPairs ? 2 : 1, *splits = c.splits, *steps_per_split = c.steps_per_split;
  return 0;
}

int tccl_weight_gradient(const tccl_weight_gradient_desc* d, void* stream) {
  const char* what = "weight_gradient";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  int rc = check_sizes(what, d->rows, d->cols, d->outputs);
  if (rc) return rc;
  if (d->dtype != TCCL_F16 && d->dtype != TCCL_BF16) return reportf(TCCL_ERR_UNSUPPORTED, "%s: grad is F16 or BF16", what);
  if (d->out_dtype != d->dtype && d->out_dtype != TCCL_F32) return reportf(TCCL_ERR_UNSUPPORTED, "%s: out is of grad's type or F32", what);
  if (!d->out) return reportf(TCCL_ERR_INVALID, "%s: out is NULL", what);
  if (d->rows) {
    if (!d->values || !d->scales || !d->grad) return reportf(TCCL_ERR_INVALID, "%s: values, scales and grad must be non-NULL", what);
    if (((uintptr_t)d->values | (uintptr_t)d->grad) & 15) return reportf(TCCL_ERR_UNSUPPORTED, "%s: values and grad must lie on 16 bytes", what);
    if (d->rows > 1 && d->ld_grad < d->outputs) return reportf(TCCL_ERR_INVALID, "%s: grad has a pitch of %lld elements for %d columns", what, (long long)d->ld_grad, d->outputs);
    const bool whole = d->outputs % 8 == 0;
    if (((d->rows > 1 || !whole) && d->ld_grad % 8) || (!whole && d->ld_grad < d->outputs))
      return reportf(TCCL_ERR_UNSUPPORTED, "%s: grad's rows must be readable in whole 16-byte vectors (outputs %d, pitch %lld)", what, d->outputs, (long long)d->ld_grad);
    if (d->ld_grad > (1ll << 24)) return reportf(TCCL_ERR_UNSUPPORTED, "%s: grad's pitch of %lld elements", what, (long long)d->ld_grad);
  }
  const int rows = d->transposed ? d->outputs : d->cols, cols = d->transposed ? d->cols : d->outputs, osize = size_of(d->out_dtype);
  if (rows > 1 && (d->ld_out < cols || (d->add && d->ld_add < cols)))
    return reportf(TCCL_ERR_INVALID, "%s: out or add has a pitch below its %d columns", what, cols);
  if (((uintptr_t)d->out | (uintptr_t)d->add) % osize) return reportf(TCCL_ERR_INVALID, "%s: out or add is not aligned to its type", what);
  int cus = 0;
  rc = compute_units(&cus);
  if (rc) return rc;
  const Cut c = choose(d->rows, d->cols, d->outputs, cus);
  WeightArgs a;
  a.values = (const uint8_t*)d->values, a.scales = (const uint8_t*)d->scales, a.grad = (const char*)d->grad;
  a.add = (const char*)d->add, a.out = (char*)d->out, a.partial = (float*)d->workspace;
  a.tokens = d->rows, a.cols = d->cols, a.outputs = d->outputs;
  a.row_blocks = (d->rows + 7) / 8;
  a.value_pitch = ((int64_t)d->cols + 127) / 128 * 1024, a.scale_pitch = ((int64_t)a.row_blocks + 15) / 16 * 16;
  a.ld_grad = d->rows > 1 ? d->ld_grad : (d->outputs + 7) / 8 * 8, a.ld_add = d->ld_add, a.ld_out = d->ld_out, a.ld_partial = partial_pitch(cols);
  a.tiles_h = c.tiles_h, a.tiles_n = c.tiles_n, a.steps = c.steps, a.splits = c.splits, a.steps_per_split = c.steps_per_split;
  a.xcds = cus % 8 ? 1 : 8, a.per_xcd = (c.tiles_h * c.tiles_n * c.splits + a.xcds - 1) / a.xcds;
  a.band = 4;  // an XCD's run of tiles is four rows of them by as many columns as its CUs give
  const bool wide = ((uintptr_t)d->out | (uintptr_t)d->add) % (4 * osize) == 0 && (rows == 1 || (d->ld_out % 4 == 0 && d->ld_add % 4 == 0));
  a.staged = d->add && wide && c.splits == 1 && d->out_dtype == TCCL_F32 && d->ld_add <= 1 << 22;
  if (c.splits > 1) {
    const int64_t need = 4 * c.splits * partial_rows(rows, cols);
    if (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need)
      return reportf(TCCL_ERR_INVALID, "%s: the workspace has %lld bytes, %lld on 16 are needed", what, (long long)d->workspace_bytes, (long long)need);
  }
  const hipStream_t st = (hipStream_t)stream;
  const bool t = d->transposed != 0;
  if (d->dtype == TCCL_BF16) return d->out_dtype == TCCL_F32 ? launch_out<__bf16, float>(a, c, t, st) : launch_out<__bf16, __bf16>(a, c, t, st);
  return d->out_dtype == TCCL_F32 ? launch_out<_Float16, float>(a, c, t, st) : launch_out<_Float16, _Float16>(a, c, t, st);
}

}  // extern "C"
