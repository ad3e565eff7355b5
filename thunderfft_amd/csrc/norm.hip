// norm.hip -- layer norm over rows: with mean and var of a row,
//   rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd,  y = xh weight + bias,
// and its gradients, with g = dy weight:
//   dx = rstd (g - mean(g) - xh mean(g xh)),  dweight = sum over rows of dy xh,
//   dbias = sum over rows of dy.
//
// A row is held in registers, so that it is read once: 4 to 64 lanes of a wave, or up to 16
// waves, with K vectors of 16 bytes a lane.  The variance is the mean square of x - mean.
// Where a row ends inside a vector, the lane takes the last V values of the row instead; those
// that belong to the lane before it are left out of the sums and stored twice alike.
//
// The backward pass goes over the rows once as well: a workgroup takes rows in turn, keeps
// their share of dweight and dbias in registers, and leaves one partial sum a column, which
// a second kernel adds up.  Every order of summation is fixed.
//
// Memory bounds both: bfloat16 32768 x 2048 takes 52 us forward (268 MB, 5.2 TB/s) and 63 us
// backward (407 MB, 6.5 TB/s, some of it still cached), 5 more for adding the parts up; half
// 2048 x 8192 14 us, 28 us and 4 us.  Few rows are bound by latency: bfloat16 8 x 1024 2.6 us,
// float 1001 x 777 4.3 us, 6.7 us and 3.3 us.  These are the kernels' own times, a training step
// of forward and backward passes in turn; further down "a call" is a backward call among its
// like, with both its kernels and the time between them (75 us at bfloat16 32768 x 2048, whose
// dy and x the forward pass has then not just brought into the caches).
#include "norm_rows.hpp"
#include "sequence.hpp"

namespace thff {
namespace {

template <class R>
__global__ __launch_bounds__(R::kLanes) void norm_forward(NormForward a) {
    using T = typename R::T;
    constexpr int V = R::V, K = R::K;
    __shared__ float lds[2][1][R::W];
    const Place<R> p;
    const long long row = static_cast<long long>(blockIdx.x) * R::kRows + threadIdx.x / R::kRowLanes;
    // Rows past the last are the last, and not stored.
    const long long r = min(row, a.rows - 1);
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    pack<T, V> in[K];
#pragma unroll
    for (int j = 0; j < K; ++j) in[j] = load_pack<T, V>(x + p.at(j, a.cols));
    float v[K][V], sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[j][i] = to_float<T>(in[j][i]);
            if (i >= p.skip(j, a.cols)) sum[0] += v[j][i];
        }
    row_sums<R>(sum, lds[0]);
    const float mean = sum[0] / a.cols;
    sum[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[j][i] -= mean;
            if (i >= p.skip(j, a.cols)) sum[0] = fmaf(v[j][i], v[j][i], sum[0]);
        }
    row_sums<R>(sum, lds[1]);
    const float rstd = 1.0f / sqrtf(sum[0] / a.cols + a.eps);
    if (row >= a.rows) return;
    T* y = static_cast<T*>(a.y) + r * a.y_stride;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int at = p.at(j, a.cols);
        const pack<float, V> w = weights_at<V>(a.weight, at, 1.0f), b = weights_at<V>(a.bias, at, 0.0f);
        pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = from_float<T>(fmaf(v[j][i] * rstd, w[i], b[i]));
        if (p.skip(j, a.cols) < V) store_pack<T, V>(y + at, out);
    }
    if (p.lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
}

template <class R>
__global__ __launch_bounds__(R::kLanes) void norm_backward(NormBackward a, int parts) {
    using T = typename R::T;
    constexpr int V = R::V, K = R::K, G = R::kRows;
    constexpr int kWaveRows = R::WPR > 1 ? 1 : 64 / R::LPR;  // rows side by side in a wave
    __shared__ float lds[2][2][R::W];
    const Place<R> p;
    const int group = threadIdx.x / R::kRowLanes;
    float dw[K][V] = {}, db[K][V] = {};
    pack<float, V> w[K];
#pragma unroll
    for (int j = 0; j < K; ++j) w[j] = weights_at<V>(a.weight, p.at(j, a.cols), 1.0f);

    struct Row {
        pack<T, V> x[K], dy[K];
        float mean, rstd;
    };
    const long long every = static_cast<long long>(parts) * G;
    const long long row0 = static_cast<long long>(blockIdx.x) * G + group;
    const auto load = [&](Row& to, long long row) {
        const long long r = min(row, a.rows - 1);
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            to.x[j] = load_pack<T, V>(x + p.at(j, a.cols));
            to.dy[j] = load_pack<T, V>(dy + p.at(j, a.cols));
        }
        to.mean = a.mean[r];
        to.rstd = a.rstd[r];
    };
    // A row past the last is the last again: its dx is stored again alike, and its share of the
    // weights' gradients left out.
    const auto take = [&](const Row& in, long long row, long long n) {
        float sums[2] = {0.0f, 0.0f};
        const bool valid = row < a.rows;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int skip = p.skip(j, a.cols), out = valid ? skip : V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (to_float<T>(in.x[j][i]) - in.mean) * in.rstd;
                const float d = to_float<T>(in.dy[j][i]), g = d * w[j][i];
                sums[0] += i >= skip ? g : 0.0f;
                sums[1] += i >= skip ? g * xh : 0.0f;
                dw[j][i] += i >= out ? d * xh : 0.0f;
                db[j][i] += i >= out ? d : 0.0f;
            }
        }
        row_sums<R>(sums, lds[n & 1]);
        const float along = sums[1] / a.cols, level = sums[0] / a.cols;
        T* dx = static_cast<T*>(a.dx) + min(row, a.rows - 1) * a.dx_stride;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            pack<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (to_float<T>(in.x[j][i]) - in.mean) * in.rstd;
                out[i] = from_float<T>(in.rstd * (to_float<T>(in.dy[j][i]) * w[j][i] - level - xh * along));
            }
            store_pack<T, V>(dx + p.at(j, a.cols), out);
        }
    };
    const long long steps = (a.rows + every - 1) / every;
    if constexpr (R::W < 16) {
        // The next row's loads are under way while a row is worked on, and go before its stores: a
        // wait for them is none for those.  Nothing in the loop branches around a load or a store,
        // so that the compiler can tell which is which.
        Row one, two;
        load(one, row0);
        for (long long n = 0; n < steps; n += 2) {
            const long long row = row0 + n * every;
            load(two, row + every);
            take(one, row, n);
            if (n + 1 == steps) break;
            load(one, row + 2 * every);
            take(two, row + every, n + 1);
        }
    } else {
        // 16 waves have 128 registers each, not enough for a second row.
        for (long long n = 0; n < steps; ++n) {
            Row one;
            load(one, row0 + n * every);
            take(one, row0 + n * every, n);
        }
    }
    if (!a.dweight && !a.dbias) return;
    // The sums of the rows side by side, then of the groups of waves, halving their number.
    constexpr int kGroups = R::W / R::WPR;
    __shared__ float others[kGroups > 1 ? kGroups / 2 : 1][K][V][kGroups > 1 ? R::kRowLanes : 1];
    const auto total = [&](float (&v)[K][V], float* to) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int m = R::LPR; m < R::LPR * kWaveRows; m *= 2) v[j][i] += __shfl_xor(v[j][i], m);
        const int part = threadIdx.x / 64 / R::WPR;
        const bool first = kWaveRows == 1 || threadIdx.x % 64 < R::LPR;
#pragma unroll
        for (int half = kGroups / 2; half > 0; half /= 2) {
            __syncthreads();
            if (first && part >= half && part < 2 * half) {
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) others[part - half][j][i][p.lane] = v[j][i];
            }
            __syncthreads();
            if (first && part < half) {
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) v[j][i] += others[part][j][i][p.lane];
            }
        }
        if (first && part == 0) {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= p.skip(j, a.cols)) to[p.at(j, a.cols) + i] = v[j][i];
        }
    };
    // workspace[0][part][column]: dweight's, workspace[1][part][column]: dbias's.
    float* to = a.workspace + static_cast<long long>(blockIdx.x) * a.cols;
    if (a.dweight) total(dw, to);
    if (a.dbias) total(db, to + static_cast<long long>(parts) * a.cols);
}

// ---- Rows too long for registers: read again for every step of the formulas. ----

template <class T>
__global__ __launch_bounds__(kLongLanes) void long_forward(NormForward a) {
    __shared__ float lds[kLongLanes / 64];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) sum += to_float<T>(x[c]);
        const float mean = block_sum(sum, lds) / a.cols;
        float square = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) {
            const float d = to_float<T>(x[c]) - mean;
            square = fmaf(d, d, square);
        }
        const float rstd = 1.0f / sqrtf(block_sum(square, lds) / a.cols + a.eps);
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) {
            const float xh = (to_float<T>(x[c]) - mean) * rstd;
            y[c] = from_float<T>(fmaf(xh, a.weight ? a.weight[c] : 1.0f, a.bias ? a.bias[c] : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

template <class T>
__global__ __launch_bounds__(kLongLanes) void long_backward(NormBackward a) {
    __shared__ float lds[kLongLanes / 64];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum = 0.0f, along = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) {
            const float g = to_float<T>(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            sum += g;
            along = fmaf(g, (to_float<T>(x[c]) - mean) * rstd, along);
        }
        sum = block_sum(sum, lds) / a.cols;
        along = block_sum(along, lds) / a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) {
            const float g = to_float<T>(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float xh = (to_float<T>(x[c]) - mean) * rstd;
            dx[c] = from_float<T>(rstd * (g - sum - xh * along));
        }
    }
}

// 32 columns a workgroup, 32 lanes a column, each every 32nd row.
template <class T>
__global__ __launch_bounds__(1024) void long_weights(NormBackward a) {
    __shared__ float lds[2][32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    for (long long c0 = 32LL * blockIdx.x; c0 < a.cols; c0 += 32LL * gridDim.x) {
        const long long c = c0 + lane;
        float w = 0.0f, b = 0.0f;
        if (c < a.cols)
            for (long long row = group; row < a.rows; row += 32) {
                const float dy = to_float<T>(static_cast<const T*>(a.dy)[row * a.dy_stride + c]);
                const float x = to_float<T>(static_cast<const T*>(a.x)[row * a.x_stride + c]);
                w = fmaf(dy, (x - a.mean[row]) * a.rstd[row], w);
                b += dy;
            }
        __syncthreads();
        lds[0][group][lane] = w;
        lds[1][group][lane] = b;
        __syncthreads();
        w = lane_sum<32>(lds[0][lane][group]);
        b = lane_sum<32>(lds[1][lane][group]);
        const long long to = c0 + group;
        if (lane == 0 && to < a.cols) {
            if (a.dweight) a.dweight[to] = w;
            if (a.dbias) a.dbias[to] = b;
        }
    }
}

template <class T>
hipError_t forward_of(const NormForward& a, hipStream_t stream) {
    hipError_t err = hipSuccess;
    const bool held = with_rows<T, false>(a.cols, [&](auto type) {
        using R = decltype(type);
        // A launch has less than 2^32 lanes.
        constexpr long long kMost = (1LL << 31) / R::kLanes * R::kRows;
        NormForward part = a;
        for (long long done = 0; done < a.rows && err == hipSuccess; done += kMost) {
            part.rows = std::min(kMost, a.rows - done);
            norm_forward<R><<<static_cast<unsigned>((part.rows + R::kRows - 1) / R::kRows), R::kLanes, 0,
                              stream>>>(part);
            err = hipGetLastError();
            part.x = static_cast<const T*>(part.x) + kMost * a.x_stride;
            part.y = static_cast<T*>(part.y) + kMost * a.y_stride;
            if (part.mean) part.mean += kMost;
            if (part.rstd) part.rstd += kMost;
        }
    });
    if (held) return err;
    long_forward<T><<<long_blocks(a.rows), kLongLanes, 0, stream>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t backward_of(const NormBackward& a, hipStream_t stream) {
    const bool weights = a.dweight || a.dbias;
    const bool held = with_rows<T, true>(a.cols, [&](auto type) {
        using R = decltype(type);
        const int parts = parts_of<R>(a.rows);
        if (parts > 0) norm_backward<R><<<parts, R::kLanes, 0, stream>>>(a, parts);
        if (weights)
            add_parts<<<dim3((a.cols + 31) / 32, 2), 1024, 0, stream>>>(a.workspace, parts, a.cols,
                                                                        a.dweight, a.dbias);
    });
    if (!held) {
        if (a.rows > 0) long_backward<T><<<long_blocks(a.rows), kLongLanes, 0, stream>>>(a);
        if (weights) long_weights<T><<<long_blocks((a.cols + 31LL) / 32), 1024, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

long long norm_workspace_bytes(long long rows, int cols) {
    // One size for all types: a type's parts are at most kMostParts, and none takes a workgroup
    // for less than one row.
    // Rows too long for registers leave no parts.
    if (cols > kMostHeld<true>) return 0;
    return 8 * std::min<long long>(kMostParts, rows) * cols;
}

hipError_t launch_layer_norm(const NormForward& a, hipStream_t stream) {
    return with_type(a.precision, [&](auto v) { return forward_of<decltype(v)>(a, stream); });
}

hipError_t launch_layer_norm_backward(const NormBackward& a, hipStream_t stream) {
    return with_type(a.precision, [&](auto v) { return backward_of<decltype(v)>(a, stream); });
}

}  // namespace thff
