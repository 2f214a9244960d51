// The thread-local error text behind nemo_last_error(), shared by the files that hold entry points.
#pragma once
#include <hip/hip_runtime.h>

namespace nemo {

// Formats the text and returns `code`, so that an entry point can `return fail(...)`.
int fail(int code, const char* fmt, ...);

}  // namespace nemo

#define HIP_TRY(expr)                                                                                                              \
    do {                                                                                                                           \
        hipError_t e_ = (expr);                                                                                                    \
        if (e_ != hipSuccess)                                                                                                      \
            return nemo::fail(NEMO_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__);            \
    } while (0)
