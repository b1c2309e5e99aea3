// The opt-in of kernels that take more than 64 KB of dynamic LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>
#include <utility>
#include <vector>

namespace eg {

// Lets `kernel` take `bytes` of dynamic LDS on the current device: the attribute belongs to a kernel on a
// device, so it is set once for each pair of them, and again after a failure.  A kernel's `bytes` never change.
inline hipError_t allow_lds(const void* kernel, int bytes) {
  static std::mutex mu;
  static std::vector<std::pair<const void*, int>> done;
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  const std::pair<const void*, int> key(kernel, dev);
  if (std::find(done.begin(), done.end(), key) != done.end()) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.push_back(key);
  return e;
}

}  // namespace eg
