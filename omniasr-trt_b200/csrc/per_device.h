// What is done once per device (a kernel's attributes belong to the device that is current when they are set).
#pragma once

#include <stdint.h>

#include <atomic>

namespace omni {

class PerDevice {
 public:
  // Calls set() (0: done) if it has not succeeded for the device yet, and gives its answer; devices past 63 are not remembered.
  template <typename F>
  int once(int device, F set) {
    const uint64_t bit = device >= 0 && device < 64 ? uint64_t(1) << device : 0;
    if (done_.load(std::memory_order_acquire) & bit) return 0;
    const int e = set();
    if (e == 0) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace omni
