// What the host side of the kernels shares.
#pragma once

#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/util/Exception.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

namespace {

inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

inline int grid_of(long items, int block, long cap) {
  return (int)std::max(1L, std::min((items + block - 1) / block, cap));
}

// Lets a kernel have more LDS than the 64 KiB that need no asking, once on
// each device; `ready` is the kernel's own, a bit a device.
template <typename Fn>
inline void allow_lds(Fn* fn, size_t bytes, std::atomic<uint64_t>& ready) {
  if (bytes <= 64 * 1024) return;
  int device = 0;
  C10_HIP_CHECK(hipGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (ready.load(std::memory_order_acquire) & bit) return;
  C10_HIP_CHECK(hipFuncSetAttribute((const void*)fn,
                                    hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)bytes));
  ready.fetch_or(bit, std::memory_order_release);
}

}  // namespace
