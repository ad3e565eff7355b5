// norm.hip -- layer norm over rows: with mean and var of a row,
//   rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd,  y = xh weight + bias,
// and its gradients, with g = dy weight:
//   dx = rstd (g - mean(g) - xh mean(g xh)),  dweight = sum over rows of dy xh,
//   dbias = sum over rows of dy.
#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {
namespace {

constexpr int kLanes = 256;
constexpr int kWaves = kLanes / 64;

// Sum over the workgroup, the same on every lane and in the same order always.
__device__ __forceinline__ float block_sum(float v, float* lds) {
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float sum = 0.0f;
    for (int w = 0; w < kWaves; ++w) sum += lds[w];
    return sum;
}

// One workgroup a row.
template <class T>
__global__ __launch_bounds__(kLanes) void norm_forward(NormForward a) {
    __shared__ float lds[kWaves];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLanes) sum += to_float(x[c]);
        const float mean = block_sum(sum, lds) / a.cols;
        float square = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLanes) {
            const float d = to_float(x[c]) - mean;
            square = fmaf(d, d, square);
        }
        const float rstd = 1.0f / sqrtf(block_sum(square, lds) / a.cols + a.eps);
        for (int c = threadIdx.x; c < a.cols; c += kLanes) {
            const float xh = (to_float(x[c]) - mean) * rstd;
            y[c] = from_float<T>(fmaf(xh, a.weight ? a.weight[c] : 1.0f, a.bias ? a.bias[c] : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

template <class T>
__global__ __launch_bounds__(kLanes) void norm_backward_rows(NormBackward a) {
    __shared__ float lds[kWaves];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum = 0.0f, along = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLanes) {
            const float g = to_float(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            sum += g;
            along = fmaf(g, (to_float(x[c]) - mean) * rstd, along);
        }
        sum = block_sum(sum, lds) / a.cols;
        along = block_sum(along, lds) / a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kLanes) {
            const float g = to_float(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float xh = (to_float(x[c]) - mean) * rstd;
            dx[c] = from_float<T>(rstd * (g - sum - xh * along));
        }
    }
}

// One workgroup a column.
template <class T>
__global__ __launch_bounds__(kLanes) void norm_backward_columns(NormBackward a) {
    __shared__ float lds[kWaves];
    const int c = blockIdx.x;
    float w = 0.0f, b = 0.0f;
    for (long long row = threadIdx.x; row < a.rows; row += kLanes) {
        const float dy = to_float(static_cast<const T*>(a.dy)[row * a.dy_stride + c]);
        const float x = to_float(static_cast<const T*>(a.x)[row * a.x_stride + c]);
        w = fmaf(dy, (x - a.mean[row]) * a.rstd[row], w);
        b += dy;
    }
    w = block_sum(w, lds);
    b = block_sum(b, lds);
    if (threadIdx.x == 0) {
        if (a.dweight) a.dweight[c] = w;
        if (a.dbias) a.dbias[c] = b;
    }
}

unsigned row_blocks(long long rows) {
    return static_cast<unsigned>(rows < 0x7fffffffLL ? rows : 0x7fffffffLL);
}

template <class T>
hipError_t launch_backward(const NormBackward& a, hipStream_t stream) {
    if (a.rows) norm_backward_rows<T><<<row_blocks(a.rows), kLanes, 0, stream>>>(a);
    if (a.dweight || a.dbias) norm_backward_columns<T><<<a.cols, kLanes, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

long long norm_workspace_bytes(long long, int) { return 0; }

hipError_t launch_layer_norm(const NormForward& a, hipStream_t stream) {
    const unsigned blocks = row_blocks(a.rows);
    if (a.precision == THFF_FLOAT)
        norm_forward<float><<<blocks, kLanes, 0, stream>>>(a);
    else if (a.precision == THFF_HALF)
        norm_forward<half_t><<<blocks, kLanes, 0, stream>>>(a);
    else
        norm_forward<bfloat_t><<<blocks, kLanes, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_layer_norm_backward(const NormBackward& a, hipStream_t stream) {
    if (a.precision == THFF_FLOAT) return launch_backward<float>(a, stream);
    if (a.precision == THFF_HALF) return launch_backward<half_t>(a, stream);
    return launch_backward<bfloat_t>(a, stream);
}

}  // namespace thff
