// Settings that a kernel needs on every device it is launched on.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace b200moe {

// Runs a setting once for each device that is current when it is asked for (again where it failed): cudaFuncSetAttribute and the like act
// on the current device alone, and a process may launch on several.  Two threads at once may both run it, which does no harm to a setting.
class PerDevice {
 public:
  template <class F>
  cudaError_t operator()(F set) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;      // devices past the 64th: every time
    if ((done_.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
    err = set();
    if (err == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
    return err;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

// Lets a kernel have `bytes` of dynamic shared memory on the current device; `done` belongs to this kernel
template <class Kernel>
inline cudaError_t allow_smem(PerDevice& done, Kernel kernel, int bytes) {
  return done([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

}  // namespace b200moe
