// What is set and looked up once per kernel and device, for handles on any
// host thread. Standard C++ only: the CUDA calls are the callers' functions.
#pragma once

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <mutex>

namespace iec {

constexpr int MAX_DEVICES = 64;

// The most dynamic shared memory that a kernel may use. It only grows: it is
// compared, set and noted under one lock, so that a thread with a smaller need
// cannot lower what another has just set.
class SmemLimit {
 public:
  // Calls set(bytes, first) unless as much was set before; `first`: nothing was.
  template <class Set>
  void raise(int device, size_t bytes, Set&& set) {
    std::atomic<size_t>& noted = noted_[device % MAX_DEVICES];
    if (noted.load(std::memory_order_acquire) > bytes) return;
    std::lock_guard<std::mutex> lock(mutex_);
    const size_t before = noted.load(std::memory_order_relaxed);
    if (before > bytes) return;
    set(bytes, before == 0);
    noted.store(bytes + 1, std::memory_order_release);
  }

 private:
  std::mutex mutex_;
  std::atomic<size_t> noted_[MAX_DEVICES] = {};  // bytes + 1
};

// How many CTAs of a kernel a device holds at once, per cluster size and 16 KB
// of shared memory; 0 where a cluster has no room. Threads that ask at once may
// each look it up; they find the same.
class Residency {
 public:
  static constexpr size_t STEP = 16 * 1024;
  template <class Find>
  int get(int device, int cluster, size_t smem, Find&& find) {
    std::atomic<int>& f = found_[device % MAX_DEVICES][cluster][std::min<size_t>(15, smem / STEP)];
    int noted = f.load(std::memory_order_relaxed);
    if (noted == 0) f.store(noted = find() + 1, std::memory_order_relaxed);
    return noted - 1;
  }

 private:
  std::atomic<int> found_[MAX_DEVICES][17][16] = {};  // CTAs + 1
};

}  // namespace iec
