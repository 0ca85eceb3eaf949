// Host: what the runtime keeps for each device of a process, asked for once a device.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace mlora {

constexpr int kDevicesKept = 64;  // devices whose answers are kept; any other is asked again at every call

// The current device, -1 where the runtime does not say.
inline int current_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return -1;
  }
  return dev;
}

// The shared memory that one kernel may be launched with: an attribute of the kernel on the
// device that is current when it is set. A failure is not kept.
class SmemLimit {
 public:
  template <typename K>
  cudaError_t raise(K kern, int bytes) {
    const int dev = current_device();
    std::atomic<int>* have = dev >= 0 && dev < kDevicesKept ? &granted_[dev] : nullptr;
    if (have != nullptr && have->load(std::memory_order_acquire) >= bytes) return cudaSuccess;
    std::lock_guard<std::mutex> lock(mu_);
    if (have != nullptr && have->load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return e;
    }
    if (have != nullptr) have->store(bytes, std::memory_order_release);
    return cudaSuccess;
  }

 private:
  std::mutex mu_;
  std::atomic<int> granted_[kDevicesKept] = {};
};

// SMs of the current device (a B200's 148 where the runtime does not say).
inline int device_sm_count() {
  static std::atomic<int> counts[kDevicesKept] = {};
  const int dev = current_device();
  std::atomic<int>* kept = dev >= 0 && dev < kDevicesKept ? &counts[dev] : nullptr;
  int n = kept != nullptr ? kept->load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  if (dev < 0 || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  if (kept != nullptr) kept->store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace mlora
