// Host-side helpers shared by the translation units of libtha4_hip.so: error reporting, device selection.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdio>
#include <string>

#include "tha4_hip.h"

namespace tha4 {

// records the calling thread's last error (tha4_last_error) and returns `code`
__attribute__((visibility("hidden"))) int fail(int code, const char* msg) noexcept;
inline int fail(int code, const std::string& msg) { return fail(code, msg.c_str()); }

// (no allocation: nothing may be thrown through a C entry point)
inline int fail_hip(const char* expr, hipError_t e) noexcept {
  char text[512];
  snprintf(text, sizeof(text), "%s: %s", expr, hipGetErrorString(e));
  return fail(THA4_ERR_HIP, text);
}

#define HIP_TRY(expr)                                                                              \
  do {                                                                                             \
    hipError_t e_ = (expr);                                                                        \
    if (e_ != hipSuccess) return fail_hip(#expr, e_);                                              \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  bool switched = false;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) == hipSuccess && prev != dev) switched = (hipSetDevice(dev) == hipSuccess);
  }
  ~DeviceGuard() {
    if (switched) (void)hipSetDevice(prev);
  }
};

// device that owns a device pointer (-1: unknown) - the stateless entry points have no handle to ask
inline int device_of(const void* p) {
  hipPointerAttribute_t a;
  if (hipPointerGetAttributes(&a, p) != hipSuccess) { (void)hipGetLastError(); return -1; }
  return a.device;
}

}  // namespace tha4
