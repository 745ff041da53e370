// Host side of copy_rows_kernel (tccl_product.h): which operands of a product are copied, and where in its workspace.
#pragma once

#include <hip/hip_runtime.h>

#include "tccl_host.h"
#include "tccl_product.h"

namespace tccl {

inline int64_t vectors(int64_t n) { return (n + 7) / 8 * 8; }
// Rows that the product kernels read where they are: on 16 bytes.  A vector that has an element of the matrix is within its memory.
inline bool on_vectors(const void* at, int64_t ld, int64_t rows) { return !((uintptr_t)at & 15) && (rows <= 1 || ld % 8 == 0); }

// Copies are laid out in a workspace one behind another; without one (at NULL) they are counted only.
struct Copies {
  CopyArgs a = {};
  char* at;
  int64_t bytes = 0;
  explicit Copies(void* workspace) : at((char*)workspace) {}
  // rows x cols from `from` on, into rows of `ld_to` elements, `to_col` elements further on in the memory of the last copy or (0) in new memory.
  const char* add(const char* from, int64_t ld_from, int64_t rows, int cols, int64_t ld_to, int64_t to_col = 0) {
    if (!to_col) last = bytes, bytes += (rows * ld_to * 2 + 255) / 256 * 256;
    CopyJob& j = a.job[a.n++];
    j.from = from, j.to = at + last + to_col * 2, j.ld_from = ld_from, j.ld_to = ld_to;
    j.cols = cols, j.per_row = (int)(vectors(cols) / 8), j.chunks = rows * j.per_row;
    const int64_t wgs = (j.chunks + 255) / 256;
    j.first_wg = all, j.wgs = (int)(wgs < 1 << 20 ? wgs : 1 << 20), all += j.wgs;
    return at + last;
  }
  template <typename T>
  int launch(const char* what, hipStream_t stream) const {
    if (!a.n) return 0;
    hipLaunchKernelGGL((copy_rows_kernel<T>), dim3((unsigned)all), dim3(256), 0, stream, a);
    return launched(what);
  }

 private:
  int64_t last = 0;
  int all = 0;  // workgroups
};

}  // namespace tccl
