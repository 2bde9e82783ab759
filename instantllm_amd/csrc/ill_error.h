// Errors of the library's translation units: `fail` keeps the message for ill_last_error() and returns the code.
#pragma once
#include <cstdarg>
#include <cstdio>

#include "../../include/ill_hip.h"

namespace illerr {
int keep(int code, const char* text) noexcept;   // (ill_engine.hip: the calling thread's message)
}

namespace {

__attribute__((format(printf, 2, 3), unused)) int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return illerr::keep(code, buf);
}

}  // namespace

#define HCK(x)                                                                                                   \
  do {                                                                                                           \
    hipError_t e_ = (x);                                                                                         \
    if (e_ != hipSuccess) return fail(ILL_E_HIP, "%s: %s (%s:%d)", #x, hipGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)
