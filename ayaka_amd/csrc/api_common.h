// What the sources of the C ABI share: error reports and small rules on arguments (api.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>

namespace ayk_api {

// Record the calling thread's last error and return `code`; clear it and return AYK_OK; either of
// them for the outcome of a launch.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int ok();
int launched(hipError_t err, const char* what);
// Whether any of these addresses is not a multiple of `to`.
bool misaligned(uintptr_t to, std::initializer_list<const void*> addresses);
// Compute units of the current device.
int compute_units();

}  // namespace ayk_api
