// per_device.hpp -- what has to be done once for every GPU.
#pragma once

#include <atomic>
#include <cstdint>

namespace kib {

// A kernel's attributes (dynamic shared memory, cluster sizes) belong to a
// device: a process that has contexts on several sets them on each.
class PerDevice {
 public:
  // Runs set(), which tells whether it succeeded, unless it has succeeded for
  // this device before.  Two threads may both run it.
  template <typename Set>
  bool once(int device, Set set) {
    if (device < 0 || device >= 64) return set();
    const uint64_t bit = uint64_t{1} << device;
    if (done_.load(std::memory_order_acquire) & bit) return true;
    if (!set()) return false;
    done_.fetch_or(bit, std::memory_order_release);
    return true;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace kib
