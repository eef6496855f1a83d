// What a process does once for every device (a kernel's attributes belong to one device).
#pragma once

#include <atomic>

namespace cb {

class PerDevice {
 public:
  // Calls set() unless it has returned for this device before.  Threads that come at the
  // same time may both call it: it has to set the same each time.
  template <typename Set>
  void once(int device, Set&& set) {
    const bool kept = device >= 0 && device < kMost;
    if (kept && done_[device].load(std::memory_order_acquire)) return;
    set();
    if (kept) done_[device].store(true, std::memory_order_release);
  }

 private:
  static constexpr int kMost = 64;
  std::atomic<bool> done_[kMost] = {};
};

}  // namespace cb
