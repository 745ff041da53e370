// Weight gradients from activations in 8 bits: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_host.h"
#include "tccl_weight.h"

namespace {

using namespace tccl;

struct Cut {
  bool large;  // 256 x 256 tiles, else 128 x 128
  int tiles_h, tiles_n, steps, splits, steps_per_split;
};

Cut cut_of(bool large, int splits, int rows, int cols, int outputs) {
  const int edge = large ? 256 : 128;
  Cut c;
  c.large = large;
  c.tiles_h = (cols + edge - 1) / edge, c.tiles_n = (outputs + edge - 1) / edge;
  c.steps = (rows + 63) / 64;
  c.steps_per_split = (c.steps + splits - 1) / splits;
  c.splits = c.steps ? (c.steps + c.steps_per_split - 1) / c.steps_per_split : 1;
  return c;
}

Cut choose(int rows, int cols, int outputs, int cus) {
  const Cut large = cut_of(true, 1, rows, cols, outputs);
  const int64_t tiles = (int64_t)large.tiles_h * large.tiles_n;
  if (tiles * 2 > cus) return large;
  const Cut small = cut_of(false, 1, rows, cols, outputs);
  const int64_t n = (int64_t)small.tiles_h * small.tiles_n;
  int splits = (int)(2 * cus / n);
  const int most = small.steps / 4;
  if (splits > most) splits = most;
  return cut_of(false, splits > 1 ? splits : 1, rows, cols, outputs);
}

int64_t partial_pitch(int cols) { return ((int64_t)cols + 3) / 4 * 4; }
int64_t partial_rows(int rows, int cols) { return (int64_t)rows * partial_pitch(cols); }

template <typename T, typename OutT, bool kTransposed>
int launch(const WeightArgs& a, const Cut& c, hipStream_t stream) {
  const dim3 wgs((unsigned)(c.tiles_h * c.tiles_n * c.splits));
  if (c.large)
    hipLaunchKernelGGL((weight_gradient_kernel<T, OutT, 256, 256, kTransposed>), wgs, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((weight_gradient_kernel<T, OutT, 128, 128, kTransposed>), wgs, dim3(256), 0, stream, a);
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
  s.splits = c.splits, s.wide = a.wide;
  const int64_t units = (int64_t)s.rows * ((s.cols + 3) / 4);
  const int64_t wgs = (units + 255) / 256;
  hipLaunchKernelGGL((weight_sum_kernel<OutT>), dim3((unsigned)(wgs < 4096 ? wgs : 4096)), dim3(256), 0, stream, s);
  return launched("weight_gradient");
}

int size_of(int dtype) { return dtype == TCCL_F32 ? 4 : dtype == TCCL_F16 || dtype == TCCL_BF16 ? 2 : 0; }

}  // namespace

extern "C" {

int64_t tccl_weight_gradient_workspace(int32_t rows, int32_t cols, int32_t outputs) {
  if (rows < 0 || cols < 1 || outputs < 1) return reportf(TCCL_ERR_INVALID, "weight_gradient: sizes %d, %d, %d", rows, cols, outputs);
  int cus = 0;
  const int rc = compute_units(&cus);
  if (rc) return -1;
  const Cut c = choose(rows, cols, outputs, cus);
  if (c.splits == 1) return 0;
  const int64_t kn = partial_rows(cols, outputs), nk = partial_rows(outputs, cols);
  return 4 * c.splits * (kn > nk ? kn : nk);
}

int tccl_weight_gradient(const tccl_weight_gradient_desc* d, void* stream) {
  const char* what = "weight_gradient";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  if (d->rows < 0 || d->cols < 1 || d->outputs < 1)
    return reportf(TCCL_ERR_INVALID, "%s: rows must not be negative, cols and outputs must be positive (got %d, %d, %d)", what, d->rows, d->cols, d->outputs);
  if (d->cols > 1 << 24 || d->outputs > 1 << 24) return reportf(TCCL_ERR_UNSUPPORTED, "%s: %d x %d outputs, at most %d of either", what, d->cols, d->outputs, 1 << 24);
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
  int rc = compute_units(&cus);
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
  // An XCD takes a patch of tiles: 4 rows of them by as many columns as its CUs give.
  a.band = 4, a.xcds = cus % 8 ? 1 : 8, a.span = cus / a.xcds;
  a.wide = ((uintptr_t)d->out | (uintptr_t)d->add) % (4 * osize) == 0 && (rows == 1 || (d->ld_out % 4 == 0 && (!d->add || d->ld_add % 4 == 0)));
  a.staged = d->add && a.wide && c.splits == 1 && d->out_dtype == TCCL_F32 && d->ld_add <= 1 << 22;
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
