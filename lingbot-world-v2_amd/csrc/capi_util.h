// Shared by the C entry points: the per-thread error message, alignment checks, device facts.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

namespace lbw {

// Sets lbw_last_error()'s message of this thread and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int hip_fail(hipError_t e, const char* what);
// Compute units of the current device.
int num_cus();

// Lets kernel `f` have `bytes` of dynamic LDS on the current device (once per device and kernel: `done` is the
// kernel's own).
struct LdsAllowed {
  std::atomic<bool> on[64] = {};
};
inline hipError_t allow_lds(const void* f, int bytes, LdsAllowed& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev >= 0 && dev < 64 && done.on[dev].load(std::memory_order_acquire)) return hipSuccess;
  e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess && dev >= 0 && dev < 64) done.on[dev].store(true, std::memory_order_release);
  return e;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool mult8(int64_t s) { return (s & 7) == 0; }

}  // namespace lbw
