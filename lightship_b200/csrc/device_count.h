// device_count.h -- a whole number that each device is asked for once.
#pragma once
#include <atomic>

namespace lsc {

constexpr int kMaxDevices = 64;

// Answers are kept by device; a query that fails leaves nothing behind and is made again the next time.
class DeviceCount {
 public:
  // What `query(&n)` says of `device` (it returns whether it succeeded); -1 where it fails.
  template <typename Query>
  int get(int device, Query query) {
    std::atomic<int>& known = counts_[device];
    const int kept = known.load(std::memory_order_relaxed);
    if (kept > 0) return kept - 1;
    int n = 0;
    if (!query(&n) || n < 0) return -1;
    known.store(n + 1, std::memory_order_relaxed);
    return n;
  }

 private:
  std::atomic<int> counts_[kMaxDevices] = {};  // the number plus one; 0: not known
};

}  // namespace lsc
