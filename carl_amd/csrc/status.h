// status.h - the C-ABI's error reporting, shared by its translation units.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/carl_amd.h"

namespace carl {

// Keeps the message for carl_last_error() of the calling thread, returns the code.
int fail(int code, const std::string& msg);

// Of a kernel launch just made.
inline int launched(const char* what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? CARL_OK : fail(CARL_ERR_RUNTIME, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace carl
