// What is found out or set up once for each device of the process, by whichever thread comes first; twice does no harm.
#pragma once
#include <atomic>
#include <cuda_runtime_api.h>

namespace oa {

constexpr int PER_DEVICE_MAX = 64;         // devices that are remembered; on others it is done again every time

// Lets `kernel` have `bytes` of dynamic shared memory on the current device.  `allowed`: the kernel's own, a bit for each device.
inline cudaError_t allow_smem(std::atomic<unsigned long long>& allowed, const void* kernel, int bytes) {
  int dev = 0;
  if (cudaError_t rc = cudaGetDevice(&dev)) return rc;
  const unsigned long long bit = dev < PER_DEVICE_MAX ? 1ull << dev : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  if (cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return rc;
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return cudaSuccess;
}

// SMs of the current device; 148 where it cannot be asked.
inline int sm_count() {
  static std::atomic<int> known[PER_DEVICE_MAX];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < PER_DEVICE_MAX && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
  if (dev < PER_DEVICE_MAX) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

}  // namespace oa
