// A kernel's opt-in to dynamic shared memory above 48 KB.  The attribute belongs to the kernel on one device, so it is set
// once for every device that launches it.  Its size is a constant of the kernel, the largest that any launch asks
// for: threads that meet here (the bindings release the GIL) set the same value, in whatever order.
#pragma once

#include <atomic>
#include <cstdint>

namespace pan {

class SmemOptIn {
 public:
  // Runs `set` unless it has succeeded for `device` before; whether the kernel may launch there.
  template <typename Set>
  bool once(int device, Set&& set) {
    if (device < 0 || device >= 64) return set();  // not remembered
    const uint64_t bit = uint64_t(1) << device;
    if (done_.load(std::memory_order_acquire) & bit) return true;
    if (!set()) return false;
    done_.fetch_or(bit, std::memory_order_release);
    return true;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

#ifdef __CUDACC__
// `opted` is the kernel's own (a static beside its launch).
template <typename K>
bool allow_smem(SmemOptIn& opted, K kernel, int bytes) {
  int device = -1;
  cudaGetDevice(&device);
  return opted.once(device, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  });
}
#endif

}  // namespace pan
