// rms_norm.hip -- root-mean-square norm over rows, after a residual's addition:
//   s = x + residual, rounded to the type of the values,
//   rstd = 1 / sqrt(mean(s^2) + eps),  xh = s rstd,  y = xh weight,
// with y in the type of the values, or in 8 bits (e4m3) with a scale for every block of columns,
// and its gradients, with g = dy weight and dsum the gradient that reaches s from elsewhere:
//   dx = rstd (g - xh mean(g xh)) + dsum,  dweight = sum over rows of dy xh.
//
// s is what the next block's residual is, so the norm is that of the rounded s, and the backward
// pass reads s alone.  Rows are held as in norm.hip, and the weights' gradients summed alike.
//
// Memory bounds both: bfloat16 32768 x 2048 takes 91 us forward (537 MB, 5.9 TB/s) and 94 us backward
// (540 MB, 5.7 TB/s), 5 more for adding the parts up; with 8 bits half 4099 x 2048 11 us (59 MB, one
// round of rows).  8 rows of 1024 take 2.8 us, their latency.
#include "block.hpp"
#include "norm_rows.hpp"

namespace thff {
namespace {

constexpr float kLargest8 = 448.0f;  // of e4m3
constexpr float kLeastScale = 1.17549435e-38f;

// Maximum over groups of N neighbouring lanes, on each of them.  (A NaN is left out.)
template <int N>
__device__ __forceinline__ float lane_max(float v) {
#pragma unroll
    for (int m = 1; m < N; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// What takes a block's largest value to the largest of e4m3, and its reciprocal.
struct Scale {
    float scale, inverse, back;
    __device__ __forceinline__ explicit Scale(float largest)
        : scale(fmaxf(largest / kLargest8, kLeastScale)), inverse(1.0f / scale), back(inverse == 0.0f ? 0.0f : scale) {}
    // v / scale to the last bit: v times the reciprocal is off by an ulp or so, which moves values that lie
    // between two of e4m3's; what is left of v corrects it (float16 4099 x 2048: 11.0 us against 10.4).  Of an
    // infinite scale (an infinite weight, or a product out of range) nothing is taken back, as 0 times it is a
    // NaN: finite values over it are 0.
    __device__ __forceinline__ float of(float v) const {
        const float q = v * inverse;
        return fmaf(fmaf(-q, back, v), inverse, q);
    }
};

// Two values in e4m3, to nearest even.
__device__ __forceinline__ unsigned bits8(float a, float b) {
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

// Stores V values in 8 bits, from the skip-th on.
template <int V>
__device__ __forceinline__ void store_8bit(unsigned char* p, const float (&v)[V], const Scale& by, int skip) {
    if constexpr (V == 1) {
        if (skip == 0) *p = static_cast<unsigned char>(bits8(by.of(v[0]), 0.0f));
    } else {
        pack<unsigned char, V> out;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const unsigned two = bits8(by.of(v[i]), by.of(v[i + 1]));
            out[i] = static_cast<unsigned char>(two);
            out[i + 1] = static_cast<unsigned char>(two >> 8);
        }
        if (skip == 0) {
            store_pack<unsigned char, V>(p, out);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i >= skip) p[i] = out[i];
        }
    }
}

// Bits8: 0 y is of type T, 1 a scale for 128 columns, 2 a scale for the row.
template <class R, bool Residual, int Bits8>
__global__ __launch_bounds__(R::kLanes) void rms_forward(RmsForward a) {
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
    if constexpr (Residual) {
        const T* residual = static_cast<const T*>(a.residual) + r * a.residual_stride;
        pack<T, V> more[K];
#pragma unroll
        for (int j = 0; j < K; ++j) more[j] = load_pack<T, V>(residual + p.at(j, a.cols));
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                in[j][i] = from_float<T>(to_float<T>(in[j][i]) + to_float<T>(more[j][i]));
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float v = to_float<T>(in[j][i]);
            if (i >= p.skip(j, a.cols)) sum[0] = fmaf(v, v, sum[0]);
        }
    row_sums<R>(sum, lds[0]);
    const float rstd = 1.0f / sqrtf(sum[0] / a.cols + a.eps);
    const bool stored = row < a.rows;
    if (stored && a.sum) {
        T* to = static_cast<T*>(a.sum) + r * a.sum_stride;
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (p.skip(j, a.cols) < V) store_pack<T, V>(to + p.at(j, a.cols), in[j]);
    }
    if (stored && a.rstd && p.lane == 0) a.rstd[row] = rstd;
    if constexpr (Bits8 == 0) {
        if (!stored) return;
        T* y = static_cast<T*>(a.y) + r * a.y_stride;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int at = p.at(j, a.cols);
            const pack<float, V> w = weights_at<V>(a.weight, at, 1.0f);
            pack<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = from_float<T>(to_float<T>(in[j][i]) * rstd * w[i]);
            if (p.skip(j, a.cols) < V) store_pack<T, V>(y + at, out);
        }
    } else {
        float v[K][V], largest[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const pack<float, V> w = weights_at<V>(a.weight, p.at(j, a.cols), 1.0f);
            largest[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[j][i] = to_float<T>(in[j][i]) * rstd * w[i];
                if (i >= p.skip(j, a.cols)) largest[j] = fmaxf(largest[j], fabsf(v[j][i]));
            }
        }
        // A row whose lanes hold less than a block at a time is one block.
        constexpr bool kOne = Bits8 == 2 || R::kRowLanes * V < 128;
        constexpr int kLanesOfBlock = kOne ? R::LPR : 128 / V;
        if constexpr (kOne) {
#pragma unroll
            for (int j = 1; j < K; ++j) largest[0] = fmaxf(largest[0], largest[j]);
        }
#pragma unroll
        for (int j = 0; j < (kOne ? 1 : K); ++j) largest[j] = lane_max<kLanesOfBlock>(largest[j]);
        if constexpr (Bits8 == 2 && R::WPR > 1) {
            const int wave = threadIdx.x / 64;
            if (threadIdx.x % 64 == 0) lds[1][0][wave] = largest[0];
            __syncthreads();
            for (int w = 0; w < R::WPR; ++w) largest[0] = fmaxf(largest[0], lds[1][0][wave / R::WPR * R::WPR + w]);
        }
        if (!stored) return;
        unsigned char* q = static_cast<unsigned char*>(a.y) + r * a.y_stride;
        const int blocks = Bits8 == 2 ? 1 : (a.cols + 127) / 128;
        float* scales = a.scales + r * blocks;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int skip = p.skip(j, a.cols);
            const Scale by(largest[kOne ? 0 : j]);
            if (skip < V) store_8bit<V>(q + p.at(j, a.cols), v[j], by, skip);
            if (kOne ? j == 0 && p.lane == 0 : p.lane % kLanesOfBlock == 0 && p.column(j) < a.cols)
                scales[kOne ? 0 : p.column(j) / 128] = by.scale;
        }
    }
}

template <class R, bool Dsum>
__global__ __launch_bounds__(R::kLanes) void rms_backward(RmsBackward a, int parts) {
    using T = typename R::T;
    constexpr int V = R::V, K = R::K, G = R::kRows;
    constexpr int kWaveRows = R::WPR > 1 ? 1 : 64 / R::LPR;  // rows side by side in a wave
    __shared__ float lds[2][1][R::W];
    const Place<R> p;
    const int group = threadIdx.x / R::kRowLanes;
    float dw[K][V] = {};
    pack<float, V> w[K];
#pragma unroll
    for (int j = 0; j < K; ++j) w[j] = weights_at<V>(a.weight, p.at(j, a.cols), 1.0f);

    struct Row {
        pack<T, V> s[K], dy[K], dsum[Dsum ? K : 1];
        float rstd;
    };
    const long long every = static_cast<long long>(parts) * G;
    const long long row0 = static_cast<long long>(blockIdx.x) * G + group;
    const auto load = [&](Row& to, long long row) {
        const long long r = min(row, a.rows - 1);
        const T* s = static_cast<const T*>(a.sum) + r * a.sum_stride;
        const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            to.s[j] = load_pack<T, V>(s + p.at(j, a.cols));
            to.dy[j] = load_pack<T, V>(dy + p.at(j, a.cols));
        }
        if constexpr (Dsum) {
            const T* dsum = static_cast<const T*>(a.dsum) + r * a.dsum_stride;
#pragma unroll
            for (int j = 0; j < K; ++j) to.dsum[j] = load_pack<T, V>(dsum + p.at(j, a.cols));
        }
        to.rstd = a.rstd[r];
    };
    // A row past the last is the last again: its dx is stored again alike, and its share of the
    // weights' gradients left out.
    const auto take = [&](const Row& in, long long row, long long n) {
        float sums[1] = {0.0f};
        const bool valid = row < a.rows;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int skip = p.skip(j, a.cols), out = valid ? skip : V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = to_float<T>(in.s[j][i]) * in.rstd;
                const float along = to_float<T>(in.dy[j][i]) * xh;
                sums[0] += i >= skip ? along * w[j][i] : 0.0f;
                dw[j][i] += i >= out ? along : 0.0f;
            }
        }
        row_sums<R>(sums, lds[n & 1]);
        const float along = sums[0] / a.cols;
        T* dx = static_cast<T*>(a.dx) + min(row, a.rows - 1) * a.dx_stride;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            pack<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = to_float<T>(in.s[j][i]) * in.rstd;
                float d = in.rstd * (to_float<T>(in.dy[j][i]) * w[j][i] - xh * along);
                if constexpr (Dsum) d += to_float<T>(in.dsum[j][i]);
                out[i] = from_float<T>(d);
            }
            store_pack<T, V>(dx + p.at(j, a.cols), out);
        }
    };
    const long long steps = (a.rows + every - 1) / every;
    if constexpr (R::W < 16) {
        // The next row's loads are under way while a row is worked on, and go before its stores.
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
    if (!a.dweight) return;
    // The sums of the rows side by side, then of the groups of waves, halving their number.
    constexpr int kGroups = R::W / R::WPR;
    __shared__ float others[kGroups > 1 ? kGroups / 2 : 1][K][V][kGroups > 1 ? R::kRowLanes : 1];
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int m = R::LPR; m < R::LPR * kWaveRows; m *= 2) dw[j][i] += __shfl_xor(dw[j][i], m);
    const int part = threadIdx.x / 64 / R::WPR;
    const bool first = kWaveRows == 1 || threadIdx.x % 64 < R::LPR;
#pragma unroll
    for (int half = kGroups / 2; half > 0; half /= 2) {
        __syncthreads();
        if (first && part >= half && part < 2 * half) {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) others[part - half][j][i][p.lane] = dw[j][i];
        }
        __syncthreads();
        if (first && part < half) {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) dw[j][i] += others[part][j][i][p.lane];
        }
    }
    // workspace[part][column]
    float* to = a.workspace + static_cast<long long>(blockIdx.x) * a.cols;
    if (first && part == 0) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i >= p.skip(j, a.cols)) to[p.at(j, a.cols) + i] = dw[j][i];
    }
}

// ---- Rows too long for registers: read again for every step of the formulas.  Waves take blocks
// of 128 columns in turn, two to a lane, the same ones in every step: what a lane reads back of the
// sums, it has written itself. ----

template <class F>
__device__ __forceinline__ void each_column(int cols, F f) {
    for (long long c = 128LL * (threadIdx.x / 64); c < cols; c += 2LL * kLongLanes) {
        const long long at = c + 2 * (threadIdx.x % 64);
        f(at, at < cols, at + 1 < cols);
    }
}

template <class T>
__global__ __launch_bounds__(kLongLanes) void long_rms_forward(RmsForward a) {
    __shared__ float lds[kLongLanes / 64];
    const int blocks = a.block == 128 ? (a.cols + 127) / 128 : 1;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* residual = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
        T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
        const auto added = [&](long long c) {
            return residual ? from_float<T>(to_float<T>(x[c]) + to_float<T>(residual[c])) : x[c];
        };
        float square = 0.0f;
        each_column(a.cols, [&](long long c, bool one, bool two) {
            const T u = one ? added(c) : T(0.0f), v = two ? added(c + 1) : T(0.0f);
            square = fmaf(to_float<T>(u), to_float<T>(u), fmaf(to_float<T>(v), to_float<T>(v), square));
            if (sum && one) sum[c] = u;
            if (sum && two) sum[c + 1] = v;
        });
        const float rstd = 1.0f / sqrtf(block_sum(square, lds) / a.cols + a.eps);
        const auto normed = [&](long long c) {
            return to_float<T>(sum ? sum[c] : added(c)) * rstd * (a.weight ? a.weight[c] : 1.0f);
        };
        if (!a.scales) {
            T* y = static_cast<T*>(a.y) + row * a.y_stride;
            each_column(a.cols, [&](long long c, bool one, bool two) {
                if (one) y[c] = from_float<T>(normed(c));
                if (two) y[c + 1] = from_float<T>(normed(c + 1));
            });
        } else {
            unsigned char* q = static_cast<unsigned char*>(a.y) + row * a.y_stride;
            float whole = 0.0f;
            if (blocks == 1) {
                each_column(a.cols, [&](long long c, bool one, bool two) {
                    whole = fmaxf(whole, fmaxf(one ? fabsf(normed(c)) : 0.0f, two ? fabsf(normed(c + 1)) : 0.0f));
                });
                whole = lane_max<64>(whole);
                __syncthreads();
                if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = whole;
                __syncthreads();
                for (int w = 0; w < kLongLanes / 64; ++w) whole = fmaxf(whole, lds[w]);
                if (threadIdx.x == 0) a.scales[row] = Scale(whole).scale;
            }
            each_column(a.cols, [&](long long c, bool one, bool two) {
                const float u = one ? normed(c) : 0.0f, v = two ? normed(c + 1) : 0.0f;
                float largest = whole;
                if (blocks > 1) {
                    largest = lane_max<64>(fmaxf(fabsf(u), fabsf(v)));
                    if (threadIdx.x % 64 == 0) a.scales[row * blocks + c / 128] = Scale(largest).scale;
                }
                const Scale by(largest);
                const unsigned both = bits8(by.of(u), by.of(v));
                if (one) q[c] = static_cast<unsigned char>(both);
                if (two) q[c + 1] = static_cast<unsigned char>(both >> 8);
            });
        }
        if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
    }
}

template <class T>
__global__ __launch_bounds__(kLongLanes) void long_rms_backward(RmsBackward a) {
    __shared__ float lds[kLongLanes / 64];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* s = static_cast<const T*>(a.sum) + row * a.sum_stride;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const T* dsum = a.dsum ? static_cast<const T*>(a.dsum) + row * a.dsum_stride : nullptr;
        T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
        const float rstd = a.rstd[row];
        float along = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes)
            along = fmaf(to_float<T>(dy[c]) * (a.weight ? a.weight[c] : 1.0f), to_float<T>(s[c]) * rstd, along);
        along = block_sum(along, lds) / a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kLongLanes) {
            const float g = to_float<T>(dy[c]) * (a.weight ? a.weight[c] : 1.0f);
            const float d = rstd * (g - to_float<T>(s[c]) * rstd * along);
            dx[c] = from_float<T>(dsum ? d + to_float<T>(dsum[c]) : d);
        }
    }
}

// 32 columns a workgroup, 32 lanes a column, each every 32nd row.
template <class T>
__global__ __launch_bounds__(1024) void long_rms_weights(RmsBackward a) {
    __shared__ float lds[32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    for (long long c0 = 32LL * blockIdx.x; c0 < a.cols; c0 += 32LL * gridDim.x) {
        const long long c = c0 + lane;
        float w = 0.0f;
        if (c < a.cols)
            for (long long row = group; row < a.rows; row += 32)
                w = fmaf(to_float<T>(static_cast<const T*>(a.dy)[row * a.dy_stride + c]),
                         to_float<T>(static_cast<const T*>(a.sum)[row * a.sum_stride + c]) * a.rstd[row], w);
        __syncthreads();
        lds[group][lane] = w;
        __syncthreads();
        w = lane_sum<32>(lds[lane][group]);
        if (lane == 0 && c0 + group < a.cols) a.dweight[c0 + group] = w;
    }
}

template <class T, bool Residual, int Bits8>
hipError_t forward_of(const RmsForward& a, hipStream_t stream) {
    hipError_t err = hipSuccess;
    const bool held = with_rows<T, false>(a.cols, [&](auto type) {
        using R = decltype(type);
        // A launch has less than 2^32 lanes.
        constexpr long long kMost = (1LL << 31) / R::kLanes * R::kRows;
        const long long blocks = a.block == 128 ? (a.cols + 127) / 128 : 1;
        RmsForward part = a;
        for (long long done = 0; done < a.rows && err == hipSuccess; done += kMost) {
            part.rows = std::min(kMost, a.rows - done);
            rms_forward<R, Residual, Bits8>
                <<<static_cast<unsigned>((part.rows + R::kRows - 1) / R::kRows), R::kLanes, 0, stream>>>(part);
            err = hipGetLastError();
            part.x = static_cast<const T*>(part.x) + kMost * a.x_stride;
            if (part.residual) part.residual = static_cast<const T*>(part.residual) + kMost * a.residual_stride;
            part.y = static_cast<char*>(part.y) + kMost * a.y_stride * static_cast<long long>(Bits8 ? 1 : sizeof(T));
            if (part.scales) part.scales += kMost * blocks;
            if (part.sum) part.sum = static_cast<T*>(part.sum) + kMost * a.sum_stride;
            if (part.rstd) part.rstd += kMost;
        }
    });
    if (held) return err;
    long_rms_forward<T><<<long_blocks(a.rows), kLongLanes, 0, stream>>>(a);
    return hipGetLastError();
}

template <class T, bool Residual>
hipError_t forward_with(const RmsForward& a, hipStream_t stream) {
    if (!a.scales) return forward_of<T, Residual, 0>(a, stream);
    return a.block == 128 ? forward_of<T, Residual, 1>(a, stream) : forward_of<T, Residual, 2>(a, stream);
}

template <class T, bool Dsum>
hipError_t backward_of(const RmsBackward& a, hipStream_t stream) {
    const bool held = with_rows<T, true>(a.cols, [&](auto type) {
        using R = decltype(type);
        const int parts = parts_of<R>(a.rows);
        if (parts > 0) rms_backward<R, Dsum><<<parts, R::kLanes, 0, stream>>>(a, parts);
        if (a.dweight)
            add_parts<<<dim3((a.cols + 31) / 32, 1), 1024, 0, stream>>>(a.workspace, parts, a.cols, a.dweight,
                                                                        nullptr);
    });
    if (!held) {
        if (a.rows > 0) long_rms_backward<T><<<long_blocks(a.rows), kLongLanes, 0, stream>>>(a);
        if (a.dweight) long_rms_weights<T><<<long_blocks((a.cols + 31LL) / 32), 1024, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

long long rms_workspace_bytes(long long rows, int cols) {
    // One size for all types, as the layer norm's; rows too long for registers leave no parts.
    if (cols > kMostHeld<true>) return 0;
    return 4 * std::min<long long>(kMostParts, rows) * cols;
}

hipError_t launch_rms_norm(const RmsForward& a, hipStream_t stream) {
    return with_type(a.precision, [&](auto v) {
        using T = decltype(v);
        return a.residual ? forward_with<T, true>(a, stream) : forward_with<T, false>(a, stream);
    });
}

hipError_t launch_rms_norm_backward(const RmsBackward& a, hipStream_t stream) {
    return with_type(a.precision, [&](auto v) {
        using T = decltype(v);
        return a.dsum ? backward_of<T, true>(a, stream) : backward_of<T, false>(a, stream);
    });
}

}  // namespace thff
