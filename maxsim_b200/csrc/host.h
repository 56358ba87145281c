// Host-side helpers shared by the library's translation units (abi.cu defines
// the ones that are not inline).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/maxsim_b200.h"

namespace maxsim {

// Records a message for maxsim_b200_last_error and returns `code`.
int fail(int code, const char* fmt, ...);

// Counts a kernel launch and turns a launch error into a status.
int launch_check(const char* what);

// SMs of the current device.
int sm_count();

#define MAXSIM_CUDA(expr)                                                         \
  do {                                                                            \
    cudaError_t e_ = (expr);                                                      \
    if (e_ != cudaSuccess)                                                        \
      return fail(MAXSIM_ECUDA, "%s failed: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

// Per-device caches are written with the same value by every thread that races
// on them, through atomics, so concurrent first calls are harmless.
constexpr int kMaxDevices = 64;

// Opt a kernel in to `smem` bytes of dynamic shared memory, once per device.
template <typename Kernel>
int ensure_smem(Kernel kern, size_t smem, std::atomic<unsigned char>* done) {
  int dev = 0;
  MAXSIM_CUDA(cudaGetDevice(&dev));
  const bool track = dev >= 0 && dev < kMaxDevices;
  if (track && done[dev].load(std::memory_order_acquire)) return MAXSIM_OK;
  MAXSIM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (track) done[dev].store(1, std::memory_order_release);
  return MAXSIM_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool valid_dtype(int dtype) {
  return dtype == MAXSIM_F32 || dtype == MAXSIM_F16 || dtype == MAXSIM_BF16;
}

}  // namespace maxsim
