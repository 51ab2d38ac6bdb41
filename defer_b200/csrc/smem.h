// The dynamic shared memory limit of kernels, set at their first launch on a
// device by whichever host thread comes first.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "common.h"

namespace defer {

// Devices on which a limit has been set. A device is entered after that, so a
// thread that finds it there may launch; threads that come at the same time set
// the limit once each.
class SmemLimit {
 public:
  // Calls set() unless the current device has been through it.
  template <class F>
  void ensure(F&& set) {
    int dev = 0;
    DEFER_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;  // devices from 64 on: at every launch
    if (done_.load(std::memory_order_acquire) & bit) return;
    set();
    done_.fetch_or(bit, std::memory_order_release);
  }
  template <class K>
  static void allow(K kernel, size_t bytes) {
    DEFER_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace defer
