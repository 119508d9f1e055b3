// What has to be done once for each device before anything else on it: attributes of kernels, which all later launches rely on.
#pragma once

#include <stdint.h>

#include <atomic>
#include <mutex>

namespace b2g {

struct OncePerDevice {
  std::atomic<uint64_t> done{0};      // bit d: device d is set up
  std::mutex mu;
};

// Calls `set` (0 = success) unless it has succeeded for this device before.  Whoever comes while another thread is at it waits: the
// callers of two streams, or of the forward and the backward pass, meet here without the interpreter's lock.
template <class F>
int once_on(OncePerDevice& once, int dev, F set) {
  if (dev < 0 || dev >= 64) return set();
  const uint64_t bit = 1ull << dev;
  if (once.done.load(std::memory_order_acquire) & bit) return 0;
  std::lock_guard<std::mutex> lock(once.mu);
  if (once.done.load(std::memory_order_relaxed) & bit) return 0;
  const int rc = set();
  if (rc == 0) once.done.fetch_or(bit, std::memory_order_release);
  return rc;
}

}  // namespace b2g
