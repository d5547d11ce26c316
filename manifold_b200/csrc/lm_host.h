// Host helpers of the language-model operators: facts about a device and a
// kernel that a call would otherwise ask the runtime for every time.
#pragma once
#include <atomic>

#include "abi.h"

namespace gfn_abi {

constexpr int LM_DEVICES = 64;

// Multiprocessors of the current device.
inline int sm_count(int* out) {
  static std::atomic<int> known[LM_DEVICES];
  int dev = 0, n = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  if (dev < LM_DEVICES) n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_status(e, "cudaDeviceGetAttribute");
    if (dev < LM_DEVICES) known[dev].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return GFN_OK;
}

// Raises a kernel's dynamic shared memory limit to `bytes`, once per device;
// `done` is that kernel's record, a bit per device.
template <class Kernel>
int shared_limit(Kernel* kernel, int bytes, std::atomic<unsigned long long>* done, const char* what) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, what);
  const unsigned long long bit = dev < LM_DEVICES ? 1ull << dev : 0ull;
  if (done->load(std::memory_order_relaxed) & bit) return GFN_OK;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_status(e, what);
  done->fetch_or(bit, std::memory_order_relaxed);
  return GFN_OK;
}

}  // namespace gfn_abi
