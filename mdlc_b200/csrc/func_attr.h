// Shared-memory limit of a kernel, set once per device and growth: the call costs about a microsecond
// of host time, which a decode step would pay for every launch.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace mdlc {

constexpr int kAttrDevices = 64;

// `seen`: a static of the call site's instantiation (one per kernel). `set` is read without the lock; limits change under it, so that
// a smaller one asked for by another thread cannot land on top of a larger one that `set` records.
struct SmemLimit {
  std::atomic<int> set[kAttrDevices] = {};
  std::mutex lock;
};
template <typename Kern>
inline cudaError_t allow_smem(SmemLimit& seen, int device, Kern* kern, int bytes) {
  const bool known = device < kAttrDevices;
  if (known && seen.set[device].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  std::lock_guard<std::mutex> hold(seen.lock);
  if (known && seen.set[device].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && known) seen.set[device].store(bytes, std::memory_order_release);
  return e;
}

}  // namespace mdlc
