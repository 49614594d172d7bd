// Setup that a kernel needs once on each device (its shared-memory limit is
// kept by the device's context, so a process that uses two devices sets it on
// both).  Nothing of CUDA in here.
#pragma once

#include <stdint.h>

#include <atomic>

namespace h3b {

class OncePerDevice {
  std::atomic<uint64_t> done_{0};  // bit: device ordinal

 public:
  // Runs `setup` unless it has succeeded (0) on device `dev` before; returns
  // its result.  Devices beyond 63 run it every time.  (Two threads may both
  // run it the first time: it only sets attributes.)
  template <class F>
  int run(int dev, F setup) {
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
    if (done_.load(std::memory_order_acquire) & bit) return 0;
    const int rc = setup();
    if (rc == 0) done_.fetch_or(bit, std::memory_order_release);
    return rc;
  }
};

}  // namespace h3b
