// Set-up that a kernel needs once on every device: its attributes (the most shared memory, cluster sizes that are not portable) belong to a device, not to the process.
#pragma once
#include <atomic>
#include <cstdint>

namespace tyr {

class OncePerDevice {
 public:
  // Runs `set` unless it has succeeded on `device` already; 0, or what it returned.  A failure is not remembered.  Several threads may come at once.
  template <typename F>
  int operator()(int device, F set) {
    const uint64_t bit = device >= 0 && device < 64 ? uint64_t{1} << device : 0;      // other numbers: at every call
    if (done_.load(std::memory_order_acquire) & bit) return 0;
    const int e = set();
    if (e == 0) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace tyr
