// Shared by the host code of the serving library: status words of kernels with bounded waits (0: none gave up), shared memory.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace cb200 {

// Lets a kernel have up to `most` bytes of dynamic shared memory; asked for once a device (the call takes as long as some of the kernels).
// One `done` for every kernel.
inline cudaError_t allow_shared_memory(std::atomic<unsigned long long>& done, const void* kernel, int most) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

int prefix_device_status(bool reset);
int logprobs_device_status(bool reset);

}  // namespace cb200
