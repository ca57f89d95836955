// Shared-memory limit of a kernel, set once per device and growth: the call costs about a microsecond
// of host time, which a decode step would pay for every launch.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace mdlc {

constexpr int kAttrDevices = 64;

// `seen`: a static of the call site's instantiation (one per kernel)
struct SmemLimit {
  std::atomic<int> set[kAttrDevices] = {};
};
template <typename Kern>
inline cudaError_t allow_smem(SmemLimit& seen, int device, Kern* kern, int bytes) {
  if (device < kAttrDevices && seen.set[device].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < kAttrDevices) {
    int was = seen.set[device].load(std::memory_order_relaxed);
    while (was < bytes && !seen.set[device].compare_exchange_weak(was, bytes, std::memory_order_relaxed)) {
    }
  }
  return e;
}

}  // namespace mdlc
