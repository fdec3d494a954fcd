// What a kernel is told once on each GPU.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

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

}  // namespace
}  // namespace b200
