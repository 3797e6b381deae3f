// Status codes of the C ABI with their thread-local message (capi.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace mvm {

// sets the calling thread's message and returns code
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// clears it and returns MVM_OK
__attribute__((visibility("hidden"))) int ok();
__attribute__((visibility("hidden"))) int hip_status(hipError_t e, const char* what);

}  // namespace mvm
