// Status codes' messages and device queries shared by the C entry points
// (defined in capi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jv {

// Records the calling thread's message and returns `code`.
__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
// JV_OK, or JV_ERR_HIP with `what` and HIP's own message.
int hip_status(hipError_t e, const char* what);
// Compute units of a device (-1: the current one); -1 if it cannot be queried.
int cu_count_of(int device);

}  // namespace jv
