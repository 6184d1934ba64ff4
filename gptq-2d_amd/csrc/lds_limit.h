// Kernels whose dynamic LDS may be all of a CU's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

namespace {

// Raises KERNEL's limit of dynamic LDS to a CU's 160 KB, once for each device (the attribute is per kernel and device).
// The kernel is a template value, not an argument: the record of the devices told belongs to the kernel then, where kernels
// with the same parameters have the same type.
template <auto KERNEL>
int allow_lds() {
  static std::atomic<uint64_t> told{0};
  int dev = 0;
  const int rc = (int)hipGetDevice(&dev);
  if (rc) return rc;
  if (dev < 64 && told.load(std::memory_order_relaxed) >> dev & 1) return 0;
  const int set = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           163840);
  if (!set && dev < 64) told.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  return set;
}

}  // namespace
