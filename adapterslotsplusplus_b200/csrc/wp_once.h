// wp_once.h -- what is set or asked once on each device.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>

namespace wp {

// A kernel's attributes and occupancy belong to a device, and a process may
// have an engine on each of several.
class PerDevice {
 public:
  // The current device's value: find()'s, which is asked again only while it
  // is 0 (a failure).
  template <typename F>
  int get(F&& find) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 0 || dev >= kDevices) return find();
    int v = known_[dev].load();
    if (v == 0) {
      v = find();
      known_[dev].store(v);
    }
    return v;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices] = {};
};

}  // namespace wp
