// The gated linear layer: argument checks, launch shapes and the entry points.
#include <hip/hip_runtime.h>

#pragma GCC visibility push(default)
#include "../../include/tileccl_hip.h"
#pragma GCC visibility pop
#include "tccl_copy.h"
#include "tccl_gated.h"

namespace {

using namespace tccl;

constexpr int64_t kMostPitch = 1 << 22;  // of an operand that is read in place: a tile's offsets have 32 bits

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

// A matrix that the elementwise parts touch: any alignment of its type, rows that do not overlap.
int check_matrix(const char* what, const char* name, const void* at, int64_t ld, int rows, int cols) {
  if (!at) return reportf(TCCL_ERR_INVALID, "%s: %s is NULL", what, name);
  if ((uintptr_t)at % 2) return reportf(TCCL_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
  if (rows > 1 && ld < cols) return reportf(TCCL_ERR_INVALID, "%s: %s has a pitch of %lld elements for %d columns", what, name, (long long)ld, cols);
  return 0;
}
// x and weight of a product of s.rows > 0 rows, from copies where the kernels cannot read them in place: rows that do not start on 16 bytes, inputs or
// halves of a weight that end within a vector.
int set_product(const char* what, const Sizes& s, const void* x, int64_t ld_x, const void* weight, int64_t ld_weight, int64_t up, int kmajor, ProductArgs& p, Copies& copies) {
  const int64_t weight_rows = kmajor ? s.outputs : s.inputs;
  int rc = check_matrix(what, "x", x, ld_x, s.rows, s.inputs);
  if (!rc) rc = check_matrix(what, "weight", weight, ld_weight, (int)weight_rows, kmajor ? s.inputs : s.outputs);
  if (rc) return rc;
  if (kmajor ? up < (s.outputs - 1) * ld_weight + s.inputs : up < s.outputs || (s.inputs > 1 && ld_weight < up + s.outputs))
    return reportf(TCCL_ERR_INVALID, "%s: the second projection's weight lies %lld elements behind the first's (pitch %lld)", what, (long long)up, (long long)ld_weight);
  const int64_t whole = vectors(s.inputs), width = vectors(s.outputs);
  p.M = s.rows, p.N = s.outputs, p.K = s.inputs;
  p.a = (const char*)x, p.lda = s.rows > 1 ? ld_x : whole;
  if (!on_vectors(x, ld_x, s.rows) || s.inputs % 8 || ld_x > kMostPitch) p.a = copies.add(p.a, ld_x, s.rows, s.inputs, whole), p.lda = whole;
  p.b = (const char*)weight, p.ldb = weight_rows > 1 ? ld_weight : kmajor ? whole : up + width;
  if (kmajor && (!on_vectors(weight, ld_weight, 2) || s.inputs % 8 || up % 8 || ld_weight > kMostPitch)) {
    p.b = copies.add((const char*)weight, ld_weight, s.outputs, s.inputs, whole);
    const char* second = copies.add((const char*)weight + up * 2, ld_weight, s.outputs, s.inputs, whole);
    up = (second - p.b) / 2, p.ldb = whole;
  } else if (!kmajor && (!on_vectors(weight, ld_weight, weight_rows) || up % 8 || p.ldb > kMostPitch)) {
    p.b = copies.add((const char*)weight, p.ldb, s.inputs, s.outputs, 2 * width);
    copies.add((const char*)weight + up * 2, p.ldb, s.inputs, s.outputs, 2 * width, width);
    up = width, p.ldb = 2 * width;
  }
  p.up = up * 2;
  return 0;
}

// The kernels: 256 and 128 tiles, and those for few rows, 16 blocks_m x 8 blocks_n outputs a workgroup.
struct Choice {
  int tile;  // 0: for few rows
  int blocks_m, blocks_n, splits;
};
constexpr int kRowsWaves = 8;

// The kernel for few rows addresses a weight by rows from its first row on, in 32 bits.
bool within_reach(int64_t inputs, int64_t outputs, int64_t ld_weight, bool kmajor) { return kmajor || (inputs * ld_weight + outputs) * 2 < 0xfffffff0ll; }

// Microseconds of a product by tiles: see choose().
double tiles_take(int tile, int64_t tiles, int steps, int cus) {
  const double rounds = (double)((tiles + cus - 1) / cus), busy = tiles < cus ? (double)tiles / cus : 1.0;
  return tile == 256 ? 6.0 + steps * rounds * (rounds > 1 ? 1.5 : 1.12 + 0.48 * busy) : 6.5 + (steps + 1) / 2 * rounds * (rounds > 1 ? 1.0 : 0.78 + 0.15 * busy);
}
// ... by 128 tiles with K split: several rounds of shorter ones may fill the device better, and each starts anew.
double split_takes(int64_t tiles, int blocks, int splits, int cus) {
  const double again = (double)((tiles * splits - 1) / cus);
  return tiles_take(128, tiles * splits, (blocks + splits - 1) / splits, cus) + (splits > 1 ? 1.0 + 3.0 * again : 0.0);
}
// ... by the kernels for few rows, of `wgs` workgroups with `turns` times 512 k each.  Narrow tiles of a weight by rows read it in pieces of 32 or 64
// bytes, at a rate of their own.
double rows_take(int blocks_m, int blocks_n, int64_t wgs, double turns, bool kmajor, double weight_bytes, int cus) {
  const double rounds = (double)((wgs + cus - 1) / cus);
  const double us = blocks_n == 2 ? 4.0 + rounds * (1.6 + 1.45 * turns) : blocks_n == 4 ? 4.0 + rounds * (2.2 + 2.3 * turns) : 6.5 + rounds * (blocks_m == 1 ? 3.3 : 3.8) * turns;
  const double reads = kmajor ? 0.0 : 4.0 + weight_bytes / (blocks_n == 2 ? 2.7e6 : blocks_n == 4 ? 4.2e6 : 6e6);
  return us > reads ? us : reads;
}
// ... of joining splits: a launch, and 16 bytes written and read for an output and split.
double join_takes(int splits, int64_t rows, int64_t outputs) { return 4.0 + splits * rows * outputs * 16 / 8e6; }

// The variant whose estimate is least.  The figures are fitted to calls of 1 .. 4000 rows, 104 .. 8192 outputs, 512 .. 8192 inputs, whose best
// variant the choice reaches within a tenth, mostly.  Inputs are split over workgroups where these would leave CUs without work
// (112 x 7168 x 104 in 128 tiles 46 us, split in 8 14.6, in narrow tiles split in 8 11).
Choice choose(int rows, int inputs, int outputs, bool kmajor, bool few, int cus) {
  Choice best = {0, 0, 0, 1};
  const int blocks = (inputs + 63) / 64;
  double least = 1e30;
  auto consider = [&](const Choice& c, double us) {
    if (c.splits > 1) us += join_takes(c.splits, rows, outputs);
    if (us < least) best = c, least = us;
  };
  auto consider_rows = [&](int m, int n) {
    const int64_t tiles = (int64_t)((rows + 16 * m - 1) / (16 * m)) * ((outputs + 8 * n - 1) / (8 * n));
    for (int splits = 1; splits <= 16 && (splits == 1 || (tiles * splits <= cus && blocks >= splits * kRowsWaves)); splits *= 2)
      consider({0, m, n, splits}, rows_take(m, n, tiles * splits, inputs / (512.0 * splits), kmajor, 4.0 * inputs * outputs, cus));
  };
  if (few) {
    // A k-major weight is read in whole lines whatever the tile.  One by rows is in tiles that are 64 outputs wide only, which many workgroups
    // gain from: 1 x 4096 x 4160 20 us split in 2, 26.5 in tiles of 32 outputs; 30 x 4096 x 1024 15.0 split in 8, 12.8 in tiles of 16 split in 4.
    const int m = kmajor && rows <= 16 ? 1 : kmajor && rows <= 32 ? 2 : 4;
    if (!kmajor && rows <= 64) consider_rows(rows <= 16 ? 1 : 2, 8);
    consider_rows(m, 2);
    consider_rows(m, 4);
    if (rows <= 64) return best;
  }
  const int64_t large = (int64_t)((rows + 255) / 256) * ((outputs + 127) / 128), small = (int64_t)((rows + 127) / 128) * ((outputs + 63) / 64);
  consider({256, 0, 0, 1}, tiles_take(256, large, blocks, cus));
  for (int splits = 1; splits <= 16 && (splits == 1 || blocks >= 4 * splits); ++splits)
    consider({128, 0, 0, splits}, split_takes(small, blocks, splits, cus));
  return best;
}

template <typename T, int kMB, int kNB, bool kBDeep>
void launch_rows(GatedArgs& a, const Choice& c, int cus, hipStream_t stream) {
  a.tiles_m = (a.p.M + 16 * kMB - 1) / (16 * kMB), a.tiles_n = (a.p.N + 8 * kNB - 1) / (8 * kNB);
  a.xcds = cus % 8 ? 1 : 8, a.per_xcd = (a.tiles_m * a.tiles_n * c.splits + a.xcds - 1) / a.xcds;
  hipLaunchKernelGGL((gated_rows_kernel<T, kMB, kNB, kRowsWaves, kBDeep>), dim3((unsigned)(a.xcds * a.per_xcd)), dim3(64 * kRowsWaves), 0, stream, a);
}
template <typename T>
int launch_few(const char* what, GatedArgs& a, const Choice& c, bool kmajor, int cus, hipStream_t stream) {
  switch (10 * c.blocks_m + c.blocks_n) {
    case 18: launch_rows<T, 1, 8, true>(a, c, cus, stream); break;
    case 28: launch_rows<T, 2, 8, true>(a, c, cus, stream); break;
    case 12: launch_rows<T, 1, 2, false>(a, c, cus, stream); break;
    case 14: launch_rows<T, 1, 4, false>(a, c, cus, stream); break;
    case 22: launch_rows<T, 2, 2, false>(a, c, cus, stream); break;
    case 24: launch_rows<T, 2, 4, false>(a, c, cus, stream); break;
    case 42: kmajor ? launch_rows<T, 4, 2, false>(a, c, cus, stream) : launch_rows<T, 4, 2, true>(a, c, cus, stream); break;
    default: kmajor ? launch_rows<T, 4, 4, false>(a, c, cus, stream) : launch_rows<T, 4, 4, true>(a, c, cus, stream); break;
  }
  return launched(what);
}

// All tiles of every split, in launches of at most 2^22 workgroups (a launch counts its threads in 32 bits); `launch` is given the grid of one.
template <typename Args, typename Launch>
int launch_tiles(const char* what, Args& a, int cus, Launch launch) {
  const int64_t items = (int64_t)a.tiles_m * a.tiles_n * a.splits, most = 1 << 22;
  if (items > 1 << 30) return reportf(TCCL_ERR_UNSUPPORTED, "%s: %lld tiles of the result", what, (long long)items);
  a.xcds = cus % 8 ? 1 : 8, a.band = 4;
  for (int64_t first = 0; first < items; first += most) {
    const int64_t n = items - first < most ? items - first : most;
    a.first = (int)first, a.items = (int)(first + n), a.per_xcd = (int)((n + a.xcds - 1) / a.xcds);
    launch(dim3((unsigned)(a.xcds * a.per_xcd)));
    const int rc = launched(what);
    if (rc) return rc;
  }
  return 0;
}

template <typename T, int kTile, bool kBackward>
int launch_tile(const char* what, GatedArgs& a, bool kmajor, int cus, hipStream_t stream) {
  a.tiles_m = (a.p.M + kTile - 1) / kTile, a.tiles_n = (a.p.N + kTile / 2 - 1) / (kTile / 2);
  return launch_tiles(what, a, cus, [&](dim3 wgs) {
    if (kmajor)
      hipLaunchKernelGGL((gated_kernel<T, kTile, false, kBackward>), wgs, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((gated_kernel<T, kTile, true, kBackward>), wgs, dim3(512), 0, stream, a);
  });
}

template <typename T, bool kBackward>
int launch(const char* what, GatedArgs& a, const Choice& c, bool kmajor, int cus, hipStream_t stream) {
  a.splits = c.splits, a.blocks_per_split = ((a.p.K + 63) / 64 + c.splits - 1) / c.splits;  // (a split may be left with nothing: it sums zeros)
  const int rc = !c.tile           ? launch_few<T>(what, a, c, kmajor, cus, stream)
                 : c.tile == 256 ? launch_tile<T, 256, kBackward>(what, a, kmajor, cus, stream)
                                 : launch_tile<T, 128, kBackward>(what, a, kmajor, cus, stream);
  if (rc || !a.partial) return rc;
  const int64_t wgs = ((int64_t)a.p.M * a.p.N + 255) / 256;
  hipLaunchKernelGGL((gated_join_kernel<T, kBackward>), dim3((unsigned)(wgs < 1 << 23 ? wgs : 1 << 23)), dim3(256), 0, stream, a);
  return launched(what);
}

// A product that is ready to be launched, and what it wants of the workspace: copies, then the sums of splits.
struct Prepared {
  GatedArgs a = {};
  Choice c = {};
  Copies copies;
  int64_t bytes = 0;
  int cus = 0;
  explicit Prepared(void* workspace) : copies(workspace) {}

  template <typename Desc>
  int of(const char* what, const Sizes& s, const Desc* d) {
    int rc = set_product(what, s, d->x, d->ld_x, d->weight, d->ld_weight, d->up, d->kmajor, a.p, copies);
    if (!rc) rc = compute_units(&cus);
    if (rc) return rc;
    c = choose(s.rows, s.inputs, s.outputs, d->kmajor, within_reach(s.inputs, s.outputs, a.p.ldb, d->kmajor), cus);
    bytes = copies.bytes;
    if (c.splits > 1) {
      a.partial = (float*)(copies.at + copies.bytes);
      bytes += 4ll * c.splits * s.rows * 2 * s.outputs;
    }
    a.activation = s.activation;
    return 0;
  }
  int enough(const char* what, const void* workspace, int64_t given) const {
    if (!bytes || (workspace && !((uintptr_t)workspace & 15) && given >= bytes)) return 0;
    return reportf(TCCL_ERR_INVALID, "%s: the workspace has %lld bytes, %lld on 16 are needed", what, (long long)given, (long long)bytes);
  }
  template <bool kBackward>
  int send(const char* what, int dtype, bool kmajor, hipStream_t stream) {
    const int rc = dtype == TCCL_BF16 ? copies.launch<__bf16>(what, stream) : copies.launch<_Float16>(what, stream);
    if (rc) return rc;
    return dtype == TCCL_BF16 ? launch<__bf16, kBackward>(what, a, c, kmajor, cus, stream) : launch<_Float16, kBackward>(what, a, c, kmajor, cus, stream);
  }
};

// How often these kernels split a sum, from `fewest` on: what the estimate says is quickest.
int least_splits(int rows, int inputs, int depth, int cus, int fewest) {
  const int64_t tiles = (int64_t)((rows + 127) / 128) * ((inputs + 127) / 128);
  const int blocks = (depth + 63) / 64;
  int best = 0;
  double least = 1e30;
  for (int splits = fewest; splits <= 16 && (splits == 1 || blocks >= 4 * splits); ++splits) {
    const double us = split_takes(tiles, blocks, splits, cus) + (splits > 1 ? join_takes(splits, rows, (inputs + 1) / 2) : 0.0);
    if (us < least) best = splits, least = us;
  }
  return best;
}
// The gradient of x by these kernels: how often the sum is split, 0 where the library's GEMM is left to make it, which is as quick where tiles
// are many or the sum is short (37 shapes of both layouts, this and the GEMM: 1000 x 1000 from 6000 24 to 25 us and 31 to 34, from 4096 21 and 19 to 25,
// from 1200 16 and 10 to 11; 1 x 4096 from 8192 15 and 14 to 19; 300 x 256 from 4096 12.6 and 7.4 to 8.6; 256 x 256 from 16384 16 and 16 to 29).
int input_grad_splits(int rows, int inputs, int depth, int cus) {
  const int64_t tiles = (int64_t)((rows + 127) / 128) * ((inputs + 127) / 128);
  const int blocks = (depth + 63) / 64;
  if (rows < 64 || tiles * 2 > cus || tiles * blocks < (blocks < 256 ? 4096 : 1024)) return 0;
  return least_splits(rows, inputs, depth, cus, 2);
}

int check_input_grad(const char* what, const tccl_gated_input_grad_desc* d) {
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  int rc = check_sizes(what, Sizes{d->rows, d->inputs, d->outputs, d->dtype, TCCL_SILU});
  if (rc || !d->rows) return rc;
  rc = check_matrix(what, "inner", d->inner, d->ld_inner, d->rows, 2 * d->outputs);
  if (!rc) rc = check_matrix(what, "weight", d->weight, d->ld_weight, d->kmajor ? 2 * d->outputs : d->inputs, d->kmajor ? d->inputs : 2 * d->outputs);
  return rc;
}
// The product's operands (of d->rows > 0 rows), from copies where they do not lie on vectors.
int set_input_grad(const tccl_gated_input_grad_desc* d, InputGradArgs& a, Copies& copies, int64_t& bytes, int& cus) {
  const int rc = compute_units(&cus);
  if (rc) return rc;
  const int depth = 2 * d->outputs;
  const int64_t whole = vectors(depth), width = vectors(d->inputs);
  ProductArgs& p = a.p;
  p.M = d->rows, p.N = d->inputs, p.K = depth, p.up = 0;
  p.a = (const char*)d->inner, p.lda = d->rows > 1 ? d->ld_inner : whole;
  if (!on_vectors(d->inner, d->ld_inner, d->rows) || depth % 8 || p.lda > kMostPitch) p.a = copies.add(p.a, d->ld_inner, d->rows, depth, whole), p.lda = whole;
  p.b = (const char*)d->weight, p.ldb = d->kmajor || d->inputs > 1 ? d->ld_weight : whole;
  if (d->kmajor ? !on_vectors(d->weight, d->ld_weight, 2) || p.ldb > kMostPitch : !on_vectors(d->weight, d->ld_weight, d->inputs) || depth % 8 || p.ldb > kMostPitch) {
    p.b = d->kmajor ? copies.add(p.b, d->ld_weight, depth, d->inputs, width) : copies.add(p.b, d->ld_weight, d->inputs, depth, whole);
    p.ldb = d->kmajor ? width : whole;
  }
  a.splits = input_grad_splits(d->rows, d->inputs, depth, cus);
  if (!a.splits) a.splits = least_splits(d->rows, d->inputs, depth, cus, 1);
  a.blocks_per_split = ((depth + 63) / 64 + a.splits - 1) / a.splits;
  a.ld_partial = ((int64_t)d->inputs + 3) / 4 * 4;
  bytes = copies.bytes + (a.splits > 1 ? 4ll * a.splits * d->rows * a.ld_partial : 0);
  a.partial = (float*)(copies.at + copies.bytes);
  return 0;
}

template <typename T>
int launch_input_grad(const char* what, InputGradArgs& a, bool kmajor, int cus, hipStream_t stream) {
  a.tiles_m = (a.p.M + 127) / 128, a.tiles_n = (a.p.N + 127) / 128;
  const int rc = launch_tiles(what, a, cus, [&](dim3 wgs) {
    if (kmajor)
      hipLaunchKernelGGL((input_grad_kernel<T, true>), wgs, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((input_grad_kernel<T, false>), wgs, dim3(512), 0, stream, a);
  });
  if (rc || a.splits == 1) return rc;
  const WeightSumArgs s = {a.partial, nullptr, a.out, a.ld_partial, 0, a.ld_out, a.p.M * a.ld_partial, a.p.M, a.p.N, a.splits};
  const int64_t sums = ((int64_t)a.p.M * ((a.p.N + 3) / 4) + 255) / 256;
  hipLaunchKernelGGL((weight_sum_kernel<T>), dim3((unsigned)(sums < 1 << 23 ? sums : 1 << 23)), dim3(256), 0, stream, s);
  return launched(what);
}

}  // namespace

extern "C" {

int64_t tccl_gated_workspace(const tccl_gated_desc* d) {
  const char* what = "gated_workspace";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what), -1;
  const Sizes s = {d->rows, d->inputs, d->outputs, d->dtype, d->activation};
  Prepared p(nullptr);
  if (check_sizes(what, s) || (s.rows && p.of(what, s, d))) return -1;
  return p.bytes;
}

int tccl_gated(const tccl_gated_desc* d, void* stream) {
  const char* what = "gated";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what);
  const Sizes s = {d->rows, d->inputs, d->outputs, d->dtype, d->activation};
  int rc = check_sizes(what, s);
  if (rc || !s.rows) return rc;
  rc = check_matrix(what, "out", d->out, d->ld_out, s.rows, s.outputs);
  if (!rc && d->kept) rc = check_matrix(what, "kept", d->kept, d->ld_kept, s.rows, 2 * s.outputs);
  Prepared p(d->workspace);
  if (!rc) rc = p.of(what, s, d);
  if (!rc) rc = p.enough(what, d->workspace, d->workspace_bytes);
  if (rc) return rc;
  p.a.out = (char*)d->out, p.a.ld_out = d->ld_out, p.a.kept = (char*)d->kept, p.a.ld_kept = d->ld_kept;
  return p.send<false>(what, d->dtype, d->kmajor, (hipStream_t)stream);
}

int tccl_gated_cut(int32_t rows, int32_t inputs, int32_t outputs, int32_t kmajor, int32_t compute_units, int32_t* tile, int32_t* tile_rows, int32_t* tile_outputs,
                   int32_t* splits) {
  const int rc = check_sizes("gated_cut", Sizes{rows, inputs, outputs, TCCL_BF16, TCCL_SILU});
  if (rc) return rc;
  if (compute_units < 1 || !tile || !tile_rows || !tile_outputs || !splits) return reportf(TCCL_ERR_INVALID, "gated_cut: %d compute units, or a NULL result", compute_units);
  const Choice c = choose(rows, inputs, outputs, kmajor != 0, true, compute_units);
  *tile = c.tile, *splits = c.splits;
  *tile_rows = c.tile ? c.tile : 16 * c.blocks_m, *tile_outputs = c.tile ? c.tile / 2 : 8 * c.blocks_n;
  return 0;
}

int64_t tccl_gated_grad_workspace(const tccl_gated_grad_desc* d) {
  const char* what = "gated_grad_workspace";
  if (!d) return reportf(TCCL_ERR_INVALID, "%s: the descriptor is NULL", what), -1;
  const Sizes s = {d->rows, d->inputs, d->outputs, d->dtype, d->activation};
  Prepared p(nullptr);
  if (check_sizes(what, s) || (s.rows && !d->kept && p.of(what, s, d))) return -1;
  return p.bytes;
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
    Prepared p(d->workspace);
    rc = p.of(what, s, d);
    if (!rc) rc = p.enough(what, d->workspace, d->workspace_bytes);
    if (rc) return rc;
    p.a.grad = (const char*)d->grad, p.a.ld_grad = d->ld_grad, p.a.inner = (char*)d->inner, p.a.ld_inner = d->ld_inner;
    return p.send<true>(what, d->dtype, d->kmajor, st);
  }
  rc = check_matrix(what, "kept", d->kept, d->ld_kept, s.rows, 2 * s.outputs);
  if (rc) return rc;
  const GatedGradArgs a = {(const char*)d->grad, (const char*)d->kept, (char*)d->inner, d->ld_grad, d->ld_kept, d->ld_inner, s.rows, s.outputs, s.activation};
  const int64_t wgs = ((int64_t)s.rows * ((s.outputs + 7) / 8) + 255) / 256;
  const dim3 grid((unsigned)(wgs < 1 << 23 ? wgs : 1 << 23));  // (a launch counts its threads in 32 bits)
  if (d->dtype == TCCL_BF16)
    hipLaunchKernelGGL((gated_grad_kernel<__bf16>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((gated_grad_kernel<_Float16>), grid, dim3(256), 0, st, a);
  return launched(what);
}

int tccl_gated_input_grad_cut(int32_t rows, int32_t inputs, int32_t outputs, int32_t compute_units, int32_t* splits) {
  const int rc = check_sizes("gated_input_grad_cut", Sizes{rows, inputs, outputs, TCCL_BF16, TCCL_SILU});
  if (rc) return rc;
  if (!splits) return reportf(TCCL_ERR_INVALID, "gated_input_grad_cut: a NULL result");
  int cus = compute_units;
  if (cus < 1 && tccl::compute_units(&cus)) return TCCL_ERR_INVALID;
  *splits = input_grad_splits(rows, inputs, 2 * outputs, cus);
  return 0;
}

int64_t tccl_gated_input_grad_workspace(const tccl_gated_input_grad_desc* d) {
  if (check_input_grad("gated_input_grad_workspace", d)) return -1;
  if (!d->rows) return 0;
  Copies copies(nullptr);
  InputGradArgs a = {};
  int64_t bytes = 0;
  int cus = 0;
  return set_input_grad(d, a, copies, bytes, cus) ? -1 : bytes;
}

int tccl_gated_input_grad(const tccl_gated_input_grad_desc* d, void* stream) {
  const char* what = "gated_input_grad";
  int rc = check_input_grad(what, d);
  if (rc || !d->rows) return rc;
  rc = check_matrix(what, "dx", d->dx, d->ld_dx, d->rows, d->inputs);
  if (rc) return rc;
  Copies copies(d->workspace);
  InputGradArgs a = {};
  int64_t bytes = 0;
  int cus = 0;
  rc = set_input_grad(d, a, copies, bytes, cus);
  if (rc) return rc;
  if (bytes && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < bytes))
    return reportf(TCCL_ERR_INVALID, "%s: the workspace has %lld bytes, %lld on 16 are needed", what, (long long)d->workspace_bytes, (long long)bytes);
  a.out = (char*)d->dx, a.ld_out = d->ld_dx;
  const hipStream_t st = (hipStream_t)stream;
  rc = d->dtype == TCCL_BF16 ? copies.launch<__bf16>(what, st) : copies.launch<_Float16>(what, st);
  if (rc) return rc;
  return d->dtype == TCCL_BF16 ? launch_input_grad<__bf16>(what, a, d->kmajor, cus, st) : launch_input_grad<_Float16>(what, a, d->kmajor, cus, st);
}

}  // extern "C"
