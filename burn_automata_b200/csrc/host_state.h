// host_state.h -- state that calls from several threads share on the host, free
// of CUDA so that it can be tested without a device.
#pragma once

#include <algorithm>
#include <cstddef>
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

// Launch plans: what a (device, context, kernel, block size, shared memory) was
// found to allow, and with it the kernel's limit of dynamic shared memory.
struct LaunchPlan {
  int device;
  const void* ctx;  // null: unknown, never found again
  const void* kernel;
  int threads;
  size_t smem;
  int per_sm;
  int sms;
};
class LaunchPlans {
 public:
  // Fills in the answer of a plan that is there.
  bool find(LaunchPlan* p) {
    std::lock_guard<std::mutex> lock(mu_);
    if (!p->ctx) return false;
    for (const LaunchPlan& k : plans_)
      if (same_kernel(k, *p) && k.threads == p->threads && k.smem == p->smem) {
        p->per_sm = k.per_sm;
        p->sms = k.sms;
        return true;
      }
    return false;
  }
  // set(limit, &plan) raises the kernel's limit and fills the plan in; the plan
  // is kept if it returns 0.  The limit only ever rises, launches planned earlier
  // with more shared memory keep theirs: one caller at a time reads the limits
  // there are, sets its own and leaves its plan.
  template <class Set>
  auto add(LaunchPlan* p, Set&& set) {
    std::lock_guard<std::mutex> lock(mu_);
    size_t limit = p->smem;
    for (const LaunchPlan& k : plans_)
      if (same_kernel(k, *p)) limit = std::max(limit, k.smem);
    const auto status = set(limit, p);
    if (status == decltype(status)(0)) plans_.push_back(*p);
    return status;
  }

 private:
  static bool same_kernel(const LaunchPlan& a, const LaunchPlan& b) {
    return a.device == b.device && a.ctx == b.ctx && a.kernel == b.kernel;
  }
  std::mutex mu_;
  std::vector<LaunchPlan> plans_;
};

}  // namespace npa
