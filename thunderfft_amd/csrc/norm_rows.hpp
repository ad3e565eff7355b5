// norm_rows.hpp -- what the norms over rows share: rows held in registers by lanes and waves, sums
// over them, the sums of a backward pass's parts, and rows too long for registers.
#pragma once

#include <algorithm>

#include "sequence_io.hpp"
#include "thunderfft/thunderfft.h"

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

// Workgroups of the backward pass at most, each with a partial sum: one a compute unit.  (Twice as
// many: 79 against 75 us a call at 32768 x 2048, 48 against 34 at 2048 x 8192, whose parts are
// then 34 MB, written and read, next to 101 MB of rows.)
constexpr int kMostParts = 256;

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

// ---- Rows too long for registers. ----

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

}  // namespace
}  // namespace thff
