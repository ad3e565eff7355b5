// sequence.hpp -- internal launch entry points of the sequence operators (the gated
// linear recurrence, scan.hip; layer norm, norm.hip) behind capi_sequence.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include "thunderfft/thunderfft.h"

namespace thff {

// A checked shape: strides filled in, in elements.
struct ScanShape {
    int precision;  // THFF_FLOAT, THFF_HALF, THFF_BFLOAT16
    bool channels_first;
    int batch, n, channels, states;
    long long x_stride, gate_stride, y_stride;
};

struct ScanForward {
    const void* x;
    const void* gate;
    const float* state_in;  // or null: zero
    const int* slots;       // or null: state row b for sequence b
    const int* lengths;     // or null: n for every sequence
    void* y;
    float* state_out;  // or null
    float* saved;      // or null
    void* workspace;
};

struct ScanBackward {
    const void* dy;
    const void* x;
    const void* gate;
    const float* saved;
    const float* dstate_out;  // or null: zero
    const int* lengths;
    void* dx;
    void* dgate;
    float* dstate_in;  // or null
    void* workspace;
};

// Bytes of `saved` and of `workspace` for a shape (0 where none is needed).
long long scan_saved_bytes(const ScanShape& shape);
long long scan_workspace_bytes(const ScanShape& shape);
// Whether the shape's grids fit one launch.
bool scan_fits(const ScanShape& shape);

hipError_t launch_gated_scan(const ScanShape& shape, const ScanForward& a, hipStream_t stream);
hipError_t launch_gated_scan_backward(const ScanShape& shape, const ScanBackward& a,
                                      hipStream_t stream);

struct NormForward {
    int precision;
    long long rows;
    int cols;
    const void* x;
    long long x_stride;
    const float* weight;  // or null: ones
    const float* bias;    // or null: zeros
    float eps;
    void* y;
    long long y_stride;
    float* mean;  // or null
    float* rstd;  // or null
};

struct NormBackward {
    int precision;
    long long rows;
    int cols;
    const void* dy;
    long long dy_stride;
    const void* x;
    long long x_stride;
    const float* mean;
    const float* rstd;
    const float* weight;  // or null: ones
    void* dx;
    long long dx_stride;
    float* dweight;  // or null
    float* dbias;    // or null
    float* workspace;
};

long long norm_workspace_bytes(long long rows, int cols);

hipError_t launch_layer_norm(const NormForward& a, hipStream_t stream);
hipError_t launch_layer_norm_backward(const NormBackward& a, hipStream_t stream);

}  // namespace thff
