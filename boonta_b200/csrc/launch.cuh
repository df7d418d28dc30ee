// Host-side launch helper of the stateless operators.
#pragma once

#include <atomic>

#include "common.cuh"

namespace bt {

// Lets `kernel` (one static `done` for each) use `bytes` of dynamic shared memory; asked of the driver once for
// each device.
template <class K>
inline int allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  BT_CUDA(cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return BT_OK;
  BT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit);
  return BT_OK;
}

}  // namespace bt
