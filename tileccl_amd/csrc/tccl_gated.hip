// The gated linear layer: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_gated.h"
#include "tccl_host.h"

namespace {

using namespace tccl;

// What the forward and the backward descriptor have in common.
struct Sizes {
  int rows, inputs, outputs, dtype, activation;
};
int check_sizes(const char* what, const Sizes& s) {
  if (s.rows < 0 || s.inputs < 1 || s.outputs < 1)
    return reportf(TCCL_ERR_INVALID, "%s: rows must not be negative, inputs and outputs must be positive (got %d, %d, %d)", what, s.rows, s.inputs, s.outputs);
  if (s.rows > TCCL_TRAINING_MAX_ROWS) return reportf(TCCL_ERR_UNSUPPORTED, "%s: rows=%d, at most %d", what, s.rows, TCCL_TRAINING_MAX_ROWS);
  if (s.inputs > TCCL_GATED_MAX_COLS || s.outputs > TCCL_GATED_MAX_COLS)
    return reportf(TCCL_ERR_UNSUPPORTED, "%s: %d inputs, %d outputs, at most %d of either", what, s.inputs, s.outputs, TCCL_GATED_MAX_COLS);
  if (s.dtype != TCCL_F16 && s.dtype != TCCL_BF16) return reportf(TCCL_ERR_UNSUPPORTED, "%s: dtype is F16 or BF16", what);
  if (s.activation < TCCL_SILU || s.activation > TCCL_RELU) return reportf(TCCL_ERR_INVALID, "%s: activation=%d is none of TCCL_SILU .. TCCL_RELU", what, s.activation);
  return 0;
}

int vectors(int n) { return (n + 7) / 8 * 8; }

// A matrix that the elementwise parts touch: any alignment of its type, rows that do not overlap.
int check_matrix(const char* what, const char* name, const void* at, int64_t ld, int rows, int cols) {
  if (!at) return reportf(TCCL_ERR_INVALID, "%s: %s is NULL", what, name);
  if ((uintptr_t)at % 2) return reportf(TCCL_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
  if (rows > 1 && ld < cols) return reportf(TCCL_ERR_INVALID, "%s: %s has a pitch of %lld elements for %d columns", what, name, (long long)ld, cols);
  return 0;
}
// An operand of the product: rows in whole 16-byte vectors, offsets within a tile in 32 bits.
int check_operand(const char* what, const char* name, const void* at, int64_t ld, int64_t rows, int cols) {
  if (!at) return reportf(TCCL_ERR_INVALID, "%s: %s is NULL", what, name);
  if (rows > 1 && ld < cols) return reportf(TCCL_ERR_INVALID, "%s: %s has a pitch of %lld elements for %d columns", what, name, (long long)ld, cols);
  if (((uintptr_t)at & 15) || (rows > 1 && (ld % 8 || ld < vectors(cols))))
    return reportf(TCCL_ERR_UNSUPPORTED, "%s: %s's rows must lie on 16 bytes and be readable in whole 16-byte vectors (%d columns, pitch %lld)", what, name, cols, (long long)ld);
  if (ld > 1 << 22) return reportf(TCCL_ERR_UNSUPPORTED, "%s: %s's pitch of %lld elements, at most %d", what, name, (long long)ld, 1 << 22);
  return 0;
}

// x and weight of a product of s.rows > 0 rows.
int set_product(const char* what, const Sizes& s, const void* x, int64_t ld_x, const void* weight, int64_t ld_weight, int64_t up, int kmajor, ProductArgs& p) {
  int rc = check_operand(what, "x", x, ld_x, s.rows, s.inputs);
  if (!rc) rc = kmajor ? check_operand(what, "weight", weight, ld_weight, s.outputs, s.inputs) : check_operand(what, "weight", weight, ld_weight, s.inputs, s.outputs);
  if (rc) return rc;
  if (up % 8 || (kmajor ? up < (s.outputs - 1) * ld_weight + s.inputs : up < s.outputs || (s.inputs > 1 && ld_weight < up + vectors(s.outputs))))
    return reportf(TCCL_ERR_UNSUPPORTED, "%s: the second projection's weight lies %lld elements behind the first's (pitch %lld)", what, (long long)up, (long long)ld_weight);
  p.a = (const char*)x, p.b = (const char*)weight;
  p.lda = s.rows > 1 ? ld_x : vectors(s.inputs);
  p.ldb = (kmajor ? s.outputs : s.inputs) > 1 ? ld_weight : kmajor ? vectors(s.inputs) : up + vectors(s.outputs);
  p.up = up * 2;
  p.M = s.rows, p.N = s.outputs, p.K = s.inputs;
  return 0;
}

template <typename T, int kTile, bool kBackward>
int launch_tile(const char* what, GatedArgs& a, bool kmajor, int cus, hipStream_t stream) {
  a.tiles_m = (a.p.M + kTile - 1) / kTile, a.tiles_n = (a.p.N + kTile / 2 - 1) / (kTile / 2);
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > 1 << 22) return reportf(TCCL_ERR_UNSUPPORTED, "%s: %lld tiles of the result", what, (long long)tiles);
  a.xcds = cus % 8 ? 1 : 8, a.per_xcd = (int)((tiles + a.xcds - 1) / a.xcds), a.band = 4;
  const dim3 wgs((unsigned)(a.xcds * a.per_xcd));
  if (kmajor)
    hipLaunchKernelGGL((gated_kernel<T, kTile, false, kBackward>), wgs, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((gated_kernel<T, kTile, true, kBackward>), wgs, dim3(512), 0, stream, a);
  return launched(what);
}

template <typename T, int kMB, int kNB>
int launch_rows(const char* what, GatedArgs& a, bool kmajor, int cus, hipStream_t stream) {
  constexpr int kWaves = 8;
  a.tiles_m = (a.p.M + 16 * kMB - 1) / (16 * kMB), a.tiles_n = (a.p.N + 8 * kNB - 1) / (8 * kNB);
  a.xcds = cus % 8 ? 1 : 8, a.per_xcd = (a.tiles_m * a.tiles_n + a.xcds - 1) / a.xcds;
  const dim3 wgs((unsigned)(a.xcds * a.per_xcd)), threads(64 * kWaves);
  if (kmajor)
    hipLaunchKernelGGL((gated_rows_kernel<T, kMB, kNB, kWaves, false>), wgs, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((gated_rows_kernel<T, kMB, kNB, kWaves, true>), wgs, threads, 0, stream, a);
  return launched(what);
}

// The kernel for few rows addresses a weight by rows from its first row on, in 32 bits.
bool within_reach(const ProductArgs& p, bool kmajor) { return kmajor || ((int64_t)p.K * p.ldb + p.N) * 2 < 0xfffffff0ll; }

// The kernels: 256 and 128 tiles, and those for few rows, 16 blocks_m x 8 blocks_n outputs a workgroup.
struct Choice {
  int tile;  // 0: for few rows
  int blocks_m, blocks_n;
};

Choice choose(const ProductArgs& p, bool kmajor, bool backward, int cus) {
  Choice c = {0, 0, 0};
  if (!backward && p.M <= 64 && within_reach(p, kmajor)) {
    c.blocks_m = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
    c.blocks_n = !kmajor && c.blocks_m < 4 ? 8 : p.N / 32 >= cus ? 4 : 2;
    return c;
  }
  // Tiles in rounds of what the device takes at a time: a step of 64 takes a large tile about 1.5 us, two small ones on a CU 1.0.
  const int64_t large = (int64_t)((p.M + 255) / 256) * ((p.N + 127) / 128), small = (int64_t)((p.M + 127) / 128) * ((p.N + 63) / 64);
  const double us_large = (double)((large + cus - 1) / cus) * 1.5, us_small = (double)((small + 2 * cus - 1) / (2 * cus)) * 1.0;
  c.tile = us_large <= us_small ? 256 : 128;
  return c;
}

template <typename T, bool kBackward>
int launch(const char* what, GatedArgs& a, bool kmajor, hipStream_t stream) {
  int cus = 0;
  const int rc = compute_units(&cus);
  if (rc) return rc;
  const Choice c = choose(a.p, kmajor, kBackward, cus);
  if constexpr (!kBackward)
    if (!c.tile) switch (10 * c.blocks_m + c.blocks_n) {
        case 12: return launch_rows<T, 1, 2>(what, a, kmajor, cus, stream);
        case 14: return launch_rows<T, 1, 4>(what, a, kmajor, cus, stream);
        case 18: return launch_rows<T, 1, 8>(what, a, kmajor, cus, stream);
        case 22: return launch_rows<T, 2, 2>(what, a, kmajor, cus, stream);
        case 24: return launch_rows<T, 2, 4>(what, a, kmajor, cus, stream);
        case 28: return launch_rows<T, 2, 8>(what, a, kmajor, cus, stream);
        case 42: return launch_rows<T, 4, 2>(what, a, kmajor, cus, stream);
        default: return launch_rows<T, 4, 4>(what, a, kmajor, cus, stream);
      }
  return c.tile == 256 ? launch_tile<T, 256, kBackward>(what, a, kmajor, cus, stream) : launch_tile<T, 128, kBackward>(what, a, kmajor, cus, stream);
}

}  // namespace

extern "C" {

int tccl_gated(const tccl_gated_desc* d, void* stream) {
  const char* what = "gated";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  const Sizes s = {d->rows, d->inputs, d->outputs, d->dtype, d->activation};
  int rc = check_sizes(what, s);
  if (rc || !s.rows) return rc;
  GatedArgs a = {};
  rc = set_product(what, s, d->x, d->ld_x, d->weight, d->ld_weight, d->up, d->kmajor, a.p);
  if (!rc) rc = check_matrix(what, "out", d->out, d->ld_out, s.rows, s.outputs);
  if (!rc && d->kept) rc = check_matrix(what, "kept", d->kept, d->ld_kept, s.rows, 2 * s.outputs);
  if (rc) return rc;
  a.out = (char*)d->out, a.ld_out = d->ld_out, a.kept = (char*)d->kept, a.ld_kept = d->ld_kept, a.activation = d->activation;
  return d->dtype == TCCL_BF16 ? launch<__bf16, false>(what, a, d->kmajor, (hipStream_t)stream) : launch<_Float16, false>(what, a, d->kmajor, (hipStream_t)stream);
}

int tccl_gated_grad(const tccl_gated_grad_desc* d, void* stream) {
  const char* what = "gated_grad";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  const Sizes s = {d->rows, d->inputs, d->outputs, d->dtype, d->activation};
  int rc = check_sizes(what, s);
  if (rc || !s.rows) return rc;
  rc = check_matrix(what, "grad", d->grad, d->ld_grad, s.rows, s.outputs);
  if (!rc) rc = check_matrix(what, "inner", d->inner, d->ld_inner, s.rows, 2 * s.outputs);
  if (rc) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (!d->kept) {
    GatedArgs a = {};
    rc = set_product(what, s, d->x, d->ld_x, d->weight, d->ld_weight, d->up, d->kmajor, a.p);
    if (rc) return rc;
    a.grad = (const char*)d->grad, a.ld_grad = d->ld_grad, a.inner = (char*)d->inner, a.ld_inner = d->ld_inner, a.activation = d->activation;
    return d->dtype == TCCL_BF16 ? launch<__bf16, true>(what, a, d->kmajor, st) : launch<_Float16, true>(what, a, d->kmajor, st);
  }
  rc = check_matrix(what, "kept", d->kept, d->ld_kept, s.rows, 2 * s.outputs);
  if (rc) return rc;
  const GatedGradArgs a = {(const char*)d->grad, (const char*)d->kept, (char*)d->inner, d->ld_grad, d->ld_kept, d->ld_inner, s.rows, s.outputs, s.activation};
  const int64_t wgs = ((int64_t)s.rows * ((s.outputs + 7) / 8) + 255) / 256;
  const dim3 grid((unsigned)(wgs < 8192 ? wgs : 8192));
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((gated_grad_kernel<__bf16>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((gated_grad_kernel<_Float16>), grid, dim3(256), 0, st, a);
  return launched(what);
}

}  // extern "C"
