// A limit that only rises: the dynamic shared memory that a kernel may ask for
// on one device. Setting it replaces the limit, and the same kernel is launched
// with different sizes by the host threads of several contexts, so check, set
// and note are one step: a thread with a smaller size must not come between
// another's set and note, or the noted limit would stay above the real one and
// every later launch of that size fail. A limit that is high enough costs one load.
#pragma once

#include <atomic>
#include <cstdint>
#include <mutex>

namespace si {

class RaisedLimit {
 public:
  // `set(bytes)` sets the real limit; it returns a status that is 0 for success.
  template <typename Set>
  auto raise(uint32_t bytes, Set&& set) -> decltype(set(bytes)) {
    if (noted_.load(std::memory_order_acquire) >= bytes) return {};
    std::lock_guard<std::mutex> lk(mu_);
    if (noted_.load(std::memory_order_relaxed) >= bytes) return {};
    const auto status = set(bytes);
    if (status == decltype(set(bytes)){}) noted_.store(bytes, std::memory_order_release);
    return status;
  }

 private:
  std::atomic<uint32_t> noted_{0};
  std::mutex mu_;
};

}  // namespace si
