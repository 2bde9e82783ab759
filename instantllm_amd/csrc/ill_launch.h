// Host side of the operators on device buffers: the current device, and launches. The includer provides `fail(code, format, ...)`.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/ill_hip.h"

namespace illp {
namespace {   // (each translation unit has its own `fail`)

// The current device is `dev` while this lives.
struct OnDevice {
  int was = -1, rc = ILL_OK;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&was) != hipSuccess) rc = fail(ILL_E_HIP, "no HIP device");
    else if (was != dev && hipSetDevice(dev) != hipSuccess) rc = fail(ILL_E_HIP, "device %d cannot be made current", dev);
    if (was == dev || rc) was = -1;
  }
  ~OnDevice() {
    if (was >= 0) hipSetDevice(was);
  }
};

// Enqueues a kernel and returns this launch's error (hipGetLastError may hold one of the program's own calls).
template <class... P>
hipError_t launch(void (*kernel)(P...), int64_t blocks, int threads, int lds, hipStream_t st, std::common_type_t<P>... args) {
  void* p[] = {&args...};
  return hipLaunchKernel((const void*)kernel, dim3(blocks), dim3(threads), p, lds, st);
}

}  // namespace
}  // namespace illp
