// Shared by the C entry points: the per-thread error message, alignment checks, device facts.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lbw {

// Sets lbw_last_error()'s message of this thread and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int hip_fail(hipError_t e, const char* what);
// Compute units of the current device.
int num_cus();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool mult8(int64_t s) { return (s & 7) == 0; }

}  // namespace lbw
