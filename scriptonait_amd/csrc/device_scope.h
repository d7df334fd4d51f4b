// The calling thread's current HIP device, set for a scope.
#pragma once
#include <hip/hip_runtime.h>

namespace llmhip {

struct Device {
  int prev = -1;
  bool ok = false;
  explicit Device(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    ok = prev == dev || hipSetDevice(dev) == hipSuccess;
    if (prev == dev) prev = -1;  // nothing to set back
  }
  ~Device() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

}  // namespace llmhip
