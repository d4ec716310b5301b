// Host helpers shared by the translation units of the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

#include "lps.h"

namespace lps {

inline bool dtype_ok(int d) { return d == LPS_DTYPE_F32 || d == LPS_DTYPE_BF16 || d == LPS_DTYPE_F16; }

// Compute units of the current device (looked up once per device; 256 when it
// cannot be).
inline int device_cus() {
  static std::atomic<int> cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int c = cus[dev].load(std::memory_order_relaxed);
  if (!c) {
    int n = 0;
    c = (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0) ? n : 256;
    cus[dev].store(c, std::memory_order_relaxed);
  }
  return c;
}

}  // namespace lps
