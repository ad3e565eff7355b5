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

// V values in one access that needs no more than the element's alignment (the hardware takes
// unaligned vectors; rows of an odd length start on any element).
template <class T, int V>
using pack = T __attribute__((ext_vector_type(V), aligned(alignof(T))));

template <class T, int V>
__device__ __forceinline__ pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const pack<T, V>*>(p);
}

// Past the caches: the next kernel's workgroups read from other L2s than the ones that wrote,
// and the lines would be written back first.  Against stores through them, us a queued call
// with all its kernels: layer norm 32768 x 2048 bfloat16 49.5 for 50.9 forward and 75.3 for 76.5
// backward; 60000 x 256 half 10.7 for 12.1 and 21.4 for 24.9; the recurrence 8 x 4096 x 2048
// bfloat16 89.2 for 92.0 and 147 for 153; half 256 x 64 x 4096, channels first, 70.9 for 69.6 and
// 118 for 122; 8 rows the same.
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, pack<T, V> v) {
    __builtin_nontemporal_store(v, reinterpret_cast<pack<T, V>*>(p));
}

// Stores the first `count` of V values.
template <class T, int V>
__device__ __forceinline__ void store_some(T* p, pack<T, V> v, int count) {
    if (count >= V) {
        store_pack<T, V>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < count) p[i] = v[i];
}

}  // namespace thff
