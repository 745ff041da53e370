// What entry points outside tccl_api.hip share with it: the text behind tccl_last_error_string() and the device's size.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

namespace tccl {

int report(int code, const char* text);  // keeps `text` for tccl_last_error_string(), returns `code`
int compute_units(int* out);             // of the current device; 0 or an error that has been reported

__attribute__((format(printf, 2, 3))) inline int reportf(int code, const char* fmt, ...) {
  char text[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  return report(code, text);
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : reportf((int)e, "HIP error in %s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

}  // namespace tccl
