// errors.hpp -- how the C ABI's entry points record a failure (defined in capi.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

namespace thff {

// Records the calling thread's last message and returns `code`.
int fail(int code, const std::string& message);

// THFF_EIO with "[ThunderFFT] <context>: <hip error string>".
int fail_hip(hipError_t err, const char* context);

}  // namespace thff
