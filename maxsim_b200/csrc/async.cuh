// Asynchronous copies of 16 or 4 bytes from global to shared memory, each thread
// waiting for its own.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace maxsim {

template <int BYTES>
__device__ __forceinline__ void copy_async(void* shared, const void* global) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(shared);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(global) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

}  // namespace maxsim
