// The shared memory that a kernel may be launched with.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace trnopt {

constexpr int kMaxDevices = 64;

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) acts on the calling thread's current device only. `done` holds,
// per device, the largest size already set for `fn`, so a process that drives several GPUs sets it on each of them.
// Sizes are set one at a time: of two threads' the smaller, set last, would stay.
inline cudaError_t smem_attr_once(const void* fn, int bytes, std::atomic<int>* done) {
  static std::mutex setting;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && done[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  const std::lock_guard<std::mutex> lock(setting);
  if (known && done[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && known) done[dev].store(bytes, std::memory_order_release);
  return e;
}

}  // namespace trnopt
