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
#include <algorithm>
#include <type_traits>

#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {
namespace {

template <int Control>
__device__ __forceinline__ float add_lanes(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), Control, 0xf, 0xf, true));
}

// Sum over groups of N neighbouring lanes, on each of them.
template <int N>
__device__ __forceinline__ float lane_sum(float v) {
    if constexpr (N > 1) v = add_lanes<0xb1>(v);   // lane ^ 1
    if constexpr (N > 2) v = add_lanes<0x4e>(v);   // lane ^ 2
    if constexpr (N > 4) v = add_lanes<0x141>(v);  // mirrored within 8
    if constexpr (N > 8) v = add_lanes<0x140>(v);  // mirrored within 16
    if constexpr (N > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (N > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// V values a vector, K vectors a lane, LPR lanes of each of WPR waves a row, in a workgroup
// of W waves.
template <class T_, int V_, int K_, int LPR_, int WPR_, int W_>
struct Rows {
    using T = T_;
    static constexpr int V = V_, K = K_, LPR = LPR_, WPR = WPR_, W = W_;
    static constexpr int kLanes = 64 * W, kRowLanes = LPR * WPR, kRows = kLanes / kRowLanes;
};

// A lane's place in its row.
template <class R>
struct Place {
    int lane;
    __device__ __forceinline__ Place() : lane(threadIdx.x % R::kRowLanes) {}
    __device__ __forceinline__ int column(int j) const { return (j * R::kRowLanes + lane) * R::V; }
    // Where vector j is read and stored, and how many of its values are not the lane's.
    __device__ __forceinline__ int at(int j, int cols) const { return min(column(j), cols - R::V); }
    __device__ __forceinline__ int skip(int j, int cols) const {
        return max(0, column(j) + R::V - cols);
    }
};

// N sums over a row's lanes, on each of them; `lds` is another one at every second call.
template <class R, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*lds)[R::W]) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane_sum<R::LPR>(v[n]);
    if constexpr (R::WPR > 1) {
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) lds[n][wave] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = 0.0f;
#pragma unroll
            for (int w = 0; w < R::WPR; ++w) v[n] += lds[n][wave / R::WPR * R::WPR + w];
        }
    }
}

template <int V>
__device__ __forceinline__ pack<float, V> weights_at(const float* p, int at, float none) {
    if (p) return load_pack<float, V>(p + at);
    pack<float, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
    return v;
}

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

// Workgroups of the backward pass at most, each with a partial sum: one a compute unit.  (Twice as
// many: 79 against 75 us a call at 32768 x 2048, 48 against 34 at 2048 x 8192, whose parts are
// then 34 MB, written and read, next to 101 MB of rows.)
constexpr int kMostParts = 256;

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

// Adds the parts of 32 columns: 32 lanes a column, each every 32nd part.
__global__ __launch_bounds__(1024) void add_parts(const float* parts, int count, int cols,
                                                  float* dweight, float* dbias) {
    __shared__ float lds[32][33];
    float* to = blockIdx.y == 0 ? dweight : dbias;
    if (!to) return;
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (c < cols) {
        const float* from = parts + static_cast<long long>(blockIdx.y) * count * cols + c;
#pragma unroll 8
        for (int k = group; k < count; k += 32) sum += from[static_cast<long long>(k) * cols];
    }
    lds[group][lane] = sum;
    __syncthreads();
    sum = lane_sum<32>(lds[lane][group]);
    if (lane == 0 && blockIdx.x * 32 + group < cols) to[blockIdx.x * 32 + group] = sum;
}

// ---- Rows too long for registers: read again for every step of the formulas. ----

constexpr int kLongLanes = 1024;

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = lane_sum<64>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kLongLanes / 64; ++w) sum += lds[w];
    return sum;
}

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

// Values a lane holds at most, and columns of the longest row that 16 waves hold: the same for all
// types.
template <bool Backward>
constexpr int kLaneValues = Backward ? 16 : 32;
template <bool Backward>
constexpr int kMostHeld = 1024 * kLaneValues<Backward>;

// Calls f with the type of row for `cols` values of T: as few lanes as hold the row in vectors of
// 16 bytes; one wave where that will do, so that no barrier is needed, and fewer vectors where its
// lanes have them to spare.  False if the row is too long for 16 waves.
//
// Forward: up to 32 values a lane, which are all that it keeps.  Backward: 16, next to the
// weights, two sums each, and the next row (2048 columns by 2 waves take 75 us a call for 32768 rows
// of bfloat16; by one wave with 32 values each, which spill, 84 us).
//
// Waves of a row are of every number that leaves few of them idle, up to 12, and of a workgroup as
// many as have registers for it backward, 8 to 12 (half 10000 x 4104, which takes 5 of 8 waves: 71
// against 90 us; 8000 x 5120: 55 against 67; 4000 x 12288, by 12 waves and not 16, which have none
// for the next row: 79 against 96.  12 where 8 would do: 12 against 10.3 us at half 2048 x 1024,
// whose rows then lie on fewer compute units, and 55.6 against 53 at 10000 x 4096).
template <class T, bool Backward, class F>
bool with_rows(int cols, F f) {
    constexpr int V = 16 / sizeof(T), M = kLaneValues<Backward> / V, W = Backward ? 8 : 4;
    const int vectors = (cols + V - 1) / V;
    if (cols < V) f(Rows<T, 1, 2, 4, 1, W>{});
    else if (vectors <= 4) f(Rows<T, V, 1, 4, 1, W>{});
    else if (vectors <= 8) f(Rows<T, V, 1, 8, 1, W>{});
    else if (vectors <= 16) f(Rows<T, V, 1, 16, 1, W>{});
    else if (vectors <= 32) f(Rows<T, V, 2, 16, 1, W>{});
    else if (vectors <= 64) f(Rows<T, V, 1, 64, 1, W>{});
    else if (vectors <= 128) f(Rows<T, V, 2, 64, 1, W>{});
    else if (M > 4 && vectors <= 256) f(Rows<T, V, M / 2, 64, 1, W>{});
    else if (vectors <= 64 * M) f(Rows<T, V, M, 64, 1, W>{});
    else if (vectors <= 128 * M) f(Rows<T, V, M, 64, 2, W>{});
    else if (vectors <= 192 * M) f(Rows<T, V, M, 64, 3, Backward ? 12 : 3>{});
    else if (vectors <= 256 * M) f(Rows<T, V, M, 64, 4, W>{});
    else if (vectors <= 320 * M) f(Rows<T, V, M, 64, 5, Backward ? 10 : 5>{});
    else if (vectors <= 384 * M) f(Rows<T, V, M, 64, 6, Backward ? 12 : 6>{});
    else if (vectors <= 512 * M) f(Rows<T, V, M, 64, 8, 8>{});
    else if (vectors <= 640 * M) f(Rows<T, V, M, 64, 10, 10>{});
    else if (vectors <= 768 * M) f(Rows<T, V, M, 64, 12, 12>{});
    else if (cols <= kMostHeld<Backward>) f(Rows<T, V, M, 64, 16, 16>{});
    else return false;
    return true;
}

template <class F>
auto with_type(int precision, F f) {
    if (precision == THFF_FLOAT) return f(float{});
    if (precision == THFF_HALF) return f(half_t{});
    return f(bfloat_t{});
}

// Workgroups of 1024 lanes, each for every so-many-th row or group of columns: a launch has less
// than 2^32 lanes.
unsigned long_blocks(long long count) {
    return static_cast<unsigned>(std::min<long long>(count, 1 << 20));
}

template <class R>
int parts_of(long long rows) {
    return static_cast<int>(std::min<long long>(kMostParts, (rows + R::kRows - 1) / R::kRows));
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
