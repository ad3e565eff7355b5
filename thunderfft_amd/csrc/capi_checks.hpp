// capi_checks.hpp -- argument checks and endings that the C ABI's entry points share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "errors.hpp"
#include "thunderfft/thunderfft.h"

namespace thff {

inline constexpr int kMostSize = 1 << 30;
// Elements of a strided buffer: byte offsets stay within 63 bits.
inline constexpr __int128 kMostSpan = static_cast<__int128>(1) << 60;

inline bool value_type(int p) { return p == THFF_FLOAT || p == THFF_HALF || p == THFF_BFLOAT16; }

inline bool aligned(const void* p, unsigned bytes) {
    return reinterpret_cast<std::uintptr_t>(p) % bytes == 0;
}

// Fills a stride of 0 in; false: rows of `length` would overlap, or the offsets overflow.
inline bool stride_of(long long given, long long length, long long rows, long long* stride) {
    *stride = given ? given : length;
    return *stride >= length && static_cast<__int128>(rows) * *stride <= kMostSpan;
}

inline unsigned element_bytes(int precision) { return precision == THFF_FLOAT ? 4 : 2; }

inline int finish(hipError_t err, hipStream_t s, bool synchronize, const char* who) {
    if (err != hipSuccess) return fail_hip(err, who);
    if (!synchronize) return THFF_OK;
    err = hipStreamSynchronize(s);
    return err == hipSuccess ? THFF_OK : fail_hip(err, who);
}

// Nothing is thrown through the C ABI (a message's allocation may fail).
template <class F>
auto guarded(F f) noexcept -> decltype(f()) {
    try {
        return f();
    } catch (...) {
        return THFF_EIO;
    }
}

}  // namespace thff
