// host.hpp -- what the files of the C ABI share: the thread's last error, the
// argument checks that set it, and the guard that makes a handle's device current.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdio>

namespace aq {

// The thread-local string behind adaptq_last_error() (c_api.cpp).
void set_error(const char *msg);
void clear_error();

inline void set_errorf(const char *fn, const char *what) {
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: %s", fn, what);
  set_error(msg);
}

inline bool require_handle(const void *h, const char *fn) {
  if (h) return true;
  set_errorf(fn, "null handle");
  return false;
}

inline bool require_pointer(const void *p, const char *fn, const char *param) {
  if (p) return true;
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: null %s", fn, param);
  set_error(msg);
  return false;
}

inline bool hip_fail(hipError_t e, const char *fn) {
  if (e == hipSuccess) return false;
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: HIP error: %s", fn, hipGetErrorString(e));
  set_error(msg);
  return true;
}

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) (void)hipSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    (void)hipGetDevice(&cur);
    if (prev >= 0 && cur != prev) (void)hipSetDevice(prev);
  }
};

}  // namespace aq
