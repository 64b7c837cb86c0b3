// sr_error.h -- the error text behind sr_last_error(), shared by the library's units.
#pragma once

#include <hip/hip_runtime.h>

namespace sr {

// Records the message of the calling thread's last failure and returns `code`.
__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);

// The same for a HIP runtime call: SR_ERR_HIP and HIP's own text.
int hip_fail(hipError_t err, const char* what);

}  // namespace sr
