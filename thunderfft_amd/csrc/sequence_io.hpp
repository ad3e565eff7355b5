// sequence_io.hpp -- element types of the sequence operators and how they are moved.
// Values are held in fp32 between a load and a store; a store rounds once, to nearest even.
#pragma once

#include <hip/hip_runtime.h>

namespace thff {

using half_t = _Float16;
using bfloat_t = __bf16;

template <class T>
__device__ __forceinline__ float to_float(T v) {
    return static_cast<float>(v);
}

template <class T>
__device__ __forceinline__ T from_float(float v) {
    return static_cast<T>(v);
}

}  // namespace thff
