// host_state.h -- state that calls from several threads share on the host, free
// of CUDA so that it can be tested without a device.
#pragma once

#include <cstdint>
#include <mutex>
#include <vector>

namespace npa {

// The last value seen of a count per device that only grows.
class Watermarks {
 public:
  // Whether `now` is above what earlier calls saw on this device; each growth is
  // reported once.
  bool grown(int device, uint64_t now) {
    std::lock_guard<std::mutex> lock(mu_);
    if (device >= int(seen_.size())) seen_.resize(size_t(device) + 1, 0);
    if (now <= seen_[device]) return false;
    seen_[device] = now;
    return true;
  }

 private:
  std::mutex mu_;
  std::vector<uint64_t> seen_;
};

}  // namespace npa
