// block.hpp -- internal launch entry points of a state space block's operators (the short
// convolution, short_conv.hip; the state space scan, state_scan.hip; root-mean-square norm,
// rms_norm.hip) behind capi_block.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include "thunderfft/thunderfft.h"

namespace thff {

// Checked shapes: strides filled in, in elements.
struct ConvShape {
    int precision;
    bool silu;
    int batch, n, channels, width, states;
    long long x_stride, y_stride;
};

struct ConvForward {
    const void* x;
    const float* weight;
    const float* bias;     // or null: zeros
    const void* state_in;  // or null: zeros
    const int* slots;      // or null: state row b for sequence b
    const int* lengths;    // or null: n for every sequence
    void* y;
    void* state_out;  // or null
};

struct ConvBackward {
    const void* dy;
    const void* x;
    const float* weight;
    const float* bias;
    const void* state_in;
    const void* dstate_out;  // or null: zeros
    const int* lengths;
    void* dx;
    float* dweight;   // or null
    float* dbias;     // or null
    void* dstate_in;  // or null
    float* workspace;
};

long long conv_workspace_bytes(const ConvShape& shape);

hipError_t launch_short_conv(const ConvShape& shape, const ConvForward& a, hipStream_t stream);
hipError_t launch_short_conv_backward(const ConvShape& shape, const ConvBackward& a,
                                      hipStream_t stream);

struct StateShape {
    int precision;
    int batch, n, channels, order, groups, states;
    long long x_stride, delta_stride, gate_stride, b_stride, c_stride, y_stride;
};

struct StateForward {
    const void* x;
    const void* delta;
    const float* a;
    const void* b;
    const void* c;
    const float* skip;        // or null: zeros
    const void* gate;         // or null: none
    const float* delta_bias;  // or null: zeros
    const float* state_in;    // or null: zeros
    const int* slots;
    const int* lengths;
    void* y;
    float* state_out;  // or null
    float* saved;      // or null
    float* workspace;
};

struct StateBackward {
    const void* dy;
    const void* x;
    const void* delta;
    const float* a;
    const void* b;
    const void* c;
    const float* skip;
    const void* gate;
    const float* delta_bias;
    const float* saved;
    const float* dstate_out;  // or null: zeros
    const int* lengths;
    void* dx;
    void* ddelta;
    float* da;
    void* db;
    void* dc;
    float* dskip;        // or null
    void* dgate;         // where there is a gate
    float* ddelta_bias;  // or null
    float* dstate_in;    // or null
    float* workspace;
};

// Bytes of `saved` and of `workspace` for a shape: of the forward pass, and enough for either.
long long state_saved_bytes(const StateShape& shape);
long long state_forward_bytes(const StateShape& shape);
long long state_workspace_bytes(const StateShape& shape);
// Whether the shape's grids fit one launch, and its buffers 63 bits.
bool state_fits(const StateShape& shape);

hipError_t launch_state_scan(const StateShape& shape, const StateForward& a, hipStream_t stream);
hipError_t launch_state_scan_backward(const StateShape& shape, const StateBackward& a,
                                      hipStream_t stream);

struct RmsForward {
    int precision;
    long long rows;
    int cols;
    const void* x;
    long long x_stride;
    const void* residual;  // or null: none
    long long residual_stride;
    const float* weight;  // or null: ones
    float eps;
    void* y;  // of the type of the values, or of 8 bits with scales
    long long y_stride;
    float* scales;  // or null: y is of the type of the values
    int block;      // columns of a scale: 128 or cols
    void* sum;      // or null
    long long sum_stride;
    float* rstd;  // or null
};

struct RmsBackward {
    int precision;
    long long rows;
    int cols;
    const void* dy;
    long long dy_stride;
    const void* sum;
    long long sum_stride;
    const float* rstd;
    const float* weight;
    const void* dsum;  // or null: zeros
    long long dsum_stride;
    void* dx;
    long long dx_stride;
    float* dweight;  // or null
    float* workspace;
};

long long rms_workspace_bytes(long long rows, int cols);

hipError_t launch_rms_norm(const RmsForward& a, hipStream_t stream);
hipError_t launch_rms_norm_backward(const RmsBackward& a, hipStream_t stream);

}  // namespace thff
