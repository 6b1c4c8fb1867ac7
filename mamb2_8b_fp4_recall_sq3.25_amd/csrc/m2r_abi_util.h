// Error reporting shared by the C-ABI entry points: a failing entry point
// returns a nonzero status and leaves a message for m2r_last_error().
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

int m2r_fail(const char* msg);
int m2r_check(hipError_t e, const char* what);

// Workgroup shape forced for the state-step kernels by m2r_set_step_shape
// (0 = automatic), encoded as waves_per_block * 16 + heads_per_wave.
int m2r_forced_step_shape();

// Whether a launch of `blocks` workgroups stays below the runtime's 2^32 threads.
inline bool m2r_grid_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }

// Lets a kernel have `bytes` of dynamic LDS, once on each device; `done` is the
// kernel's own, a bit for each of the first 64 devices.
inline int m2r_allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (int rc = m2r_check(hipGetDevice(&device), "device")) return rc;
  const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  if (int rc = m2r_check(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "LDS size")) return rc;
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}
