// What a kernel is told, or a GPU is asked, once on each GPU.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>

namespace b200 {
namespace {

// Runs `set` (attributes of one kernel: they belong to a device, and setting them takes the host half a microsecond) when the current device has not seen it
// yet; false where that fails.  Threads that meet set the same twice.
template <typename F> bool once_per_device(std::atomic<uint64_t>& done, F set) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); return false; }
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (!set()) { cudaGetLastError(); return false; }
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// What `find` says of the current device, which is asked once on each (beyond the 64th every time).
template <typename V> class PerDevice {
  std::mutex asking_;
  std::atomic<uint64_t> known_{0};
  V values_[64];

 public:
  template <typename F> V operator()(F find) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); return find(); }
    if (device >= 64) return find();
    if (!(known_.load(std::memory_order_acquire) >> device & 1)) {
      const std::lock_guard<std::mutex> lock(asking_);
      if (!(known_.load(std::memory_order_relaxed) >> device & 1)) {
        values_[device] = find();
        known_.fetch_or(1ull << device, std::memory_order_release);
      }
    }
    return values_[device];
  }
};

}  // namespace
}  // namespace b200
