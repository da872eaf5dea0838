// Settings that a kernel needs once on each device, made by whichever host threads call first.
#pragma once

#include <atomic>
#include <cstdint>

namespace arb {

// Several threads may run it at once, for one device or several: `set` may then run more than once on a
// device, and a device counts as done only after a `set` that returned 0 there. Devices from 64 on are set
// at every call.
class DeviceOnce {
 public:
  template <typename Set>
  auto run(int device, Set&& set) -> decltype(set()) {
    const uint64_t bit = device >= 0 && device < 64 ? uint64_t{1} << device : 0;
    using Status = decltype(set());
    if (done_.load(std::memory_order_acquire) & bit) return Status{};
    const Status status = set();
    if (status == Status{}) done_.fetch_or(bit, std::memory_order_release);
    return status;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace arb
