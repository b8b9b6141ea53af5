// smem_limits.h - which limit of dynamic shared memory each kernel has on each
// device, so that it is set once and never lowered.
#pragma once

#include <map>
#include <mutex>
#include <utility>

namespace i8c {

class SmemLimits {
 public:
  // Raises the limit of `kernel` on `device` to `bytes` through set(bytes) -> bool
  // unless it is that high already.  Any number of kernels, from any thread.
  template <class Set>
  bool ensure(int device, const void *kernel, int bytes, Set set) {
    try {
      std::lock_guard<std::mutex> lock(mutex_);
      int &limit = limits_[std::make_pair(device, kernel)];
      if (limit >= bytes) return true;
      if (!set(bytes)) return false;
      limit = bytes;
      return true;
    } catch (...) {
      return false;   // no memory for the entry; no exception leaves a C entry point
    }
  }

 private:
  std::mutex mutex_;
  std::map<std::pair<int, const void *>, int> limits_;
};

}  // namespace i8c
