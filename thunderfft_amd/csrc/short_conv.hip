// short_conv.hip -- short causal convolution per channel, K = 2 to 4 taps: with xe the K - 1 values
// of the state and then x,
//   p[t] = bias + sum_k weight[k] xe[t + k],  y[t] = p silu'd or p,
// and its gradients: dp[t] = dy[t] slope(p[t]),
//   dxe[e] = sum_k weight[k] dp[e - k]  (+ dstate_out behind the end),
//   dweight[k] = sum_t dp[t] xe[t + k],  dbias = sum_t dp[t].
//
// A lane takes 16 bytes of channels (backward 2 or 4 of them) and some steps one after the other, with the last
// K - 1 rows in registers, so that a row is read once but for those before a lane's first step.
//
// Memory bounds it: bfloat16 8 x 4096 x 2048, 4 taps, 46 us forward (294 MB, 6.4 TB/s) and 76 us
// backward (417 MB, 5.5 TB/s; the VALU issues in 90% of the cycles too), 5 more for the weights'
// sums.  A token of 8 sequences 5 us, half 7 x 1000 x 2048 of unlike lengths 12 us: a round of
// loads and one of stores.
#include <algorithm>
#include <type_traits>

#include "block.hpp"
#include "sequence_io.hpp"

namespace thff {
namespace {

constexpr int kLanes = 256;

__device__ __forceinline__ int length_of(const int* lengths, int b, int n) {
    return lengths ? min(max(lengths[b], 0), n) : n;
}

// 1 / (1 + exp(-v))
__device__ __forceinline__ float opened(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}

// v rounded to T.  (half)(a * b) may become one instruction that rounds the exact product once, or two with
// one to fp32 between; which, differs from step to step of a tile, and one in 2^14 values with it.  Held in a
// register v is fp32 everywhere, so that a sequence has the same bits however it is cut into calls.
template <class T>
__device__ __forceinline__ T rounded(float v) {
    if constexpr (std::is_same_v<T, half_t>) asm("" : "+v"(v));
    return from_float<T>(v);
}

// Where a lane's V channels are: the last lane of a row takes the last V, `skip` of which are also
// the lane's before it.
struct Channels {
    int at, skip;
};

template <int V>
__device__ __forceinline__ Channels channels_of(int vector, int channels) {
    return {min(vector * V, channels - V), max(0, vector * V + V - channels)};
}

// Stores values from the skip-th on: where the lane before stores its own, and may have read other
// values for them (states kept in place).
template <class T, int V>
__device__ __forceinline__ void store_own(T* p, pack<T, V> v, int skip) {
    if (skip == 0) {
        store_pack<T, V>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i >= skip) p[i] = v[i];
}

// w[k][i]: tap k of channel i; and the bias.
template <int V, int K>
struct Taps {
    float w[K][V], bias[V];

    __device__ __forceinline__ Taps(const float* weight, const float* b, int at) {
        const pack<float, V * K> all = load_pack<float, V * K>(weight + static_cast<long long>(at) * K);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) w[k][i] = all[i * K + k];
#pragma unroll
        for (int i = 0; i < V; ++i) bias[i] = b ? b[at + i] : 0.0f;
    }
};

// Steps of a lane forward: bfloat16 8 x 4096 x 2048 47 us, 52 by 8, 63 by 32 (registers); 1 x 65536 x
// 1024 49, 55 and 46; half 7 x 1000 x 2048 of unlike lengths 12.1, 11.7 and 14.3.
constexpr int kSteps = 16;

template <class T, int V, int K, bool Silu, int TS>
__global__ __launch_bounds__(kLanes) void conv_forward(ConvShape s, ConvForward a, int vectors, long long tiles) {
    constexpr int H = K - 1;
    const long long lanes = s.batch * tiles * vectors;
    for (long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x; i < lanes;
         i += static_cast<long long>(gridDim.x) * kLanes) {
        const long long column = i / vectors;
        const Channels c = channels_of<V>(static_cast<int>(i - column * vectors), s.channels);
        const int b = static_cast<int>(column / tiles), t0 = static_cast<int>(column - b * tiles) * TS;
        const int length = length_of(a.lengths, b, s.n);
        const T* x = static_cast<const T*>(a.x) + b * static_cast<long long>(s.n) * s.x_stride + c.at;
        if (t0 > 0 && t0 >= length) {
            T* y = static_cast<T*>(a.y) + (b * static_cast<long long>(s.n) + t0) * s.y_stride + c.at;
            for (int j = 0; j < TS && t0 + j < s.n; ++j) store_pack<T, V>(y + j * s.y_stride, pack<T, V>{});
            continue;
        }
        const Taps<V, K> taps(a.weight, a.bias, c.at);
        pack<T, V> in[TS + H];
        int slot = b;
        if (t0 == 0) {
            if (a.slots) slot = a.slots[b];
            if (a.slots && (slot < 0 || slot >= s.states)) slot = -1;
            const T* state = static_cast<const T*>(a.state_in) + static_cast<long long>(slot) * H * s.channels + c.at;
#pragma unroll
            for (int k = 0; k < H; ++k) {
                in[k] = pack<T, V>{};
                if (a.state_in && slot >= 0) in[k] = load_pack<T, V>(state + static_cast<long long>(k) * s.channels);
            }
        } else {
#pragma unroll
            for (int k = 0; k < H; ++k) in[k] = load_pack<T, V>(x + (t0 - H + k) * s.x_stride);
        }
        T* y = static_cast<T*>(a.y) + b * static_cast<long long>(s.n) * s.y_stride + c.at + t0 * s.y_stride;
        const bool whole = t0 + TS <= s.n;
        if (whole) {
            const T* from = x + t0 * s.x_stride;
#pragma unroll
            for (int j = 0; j < TS; ++j) in[H + j] = load_pack<T, V>(from + j * s.x_stride);
        } else if (s.n > 0) {
#pragma unroll
            for (int j = 0; j < TS; ++j) in[H + j] = load_pack<T, V>(x + min(t0 + j, s.n - 1) * s.x_stride);
        }
        if (t0 == 0 && a.state_out && slot >= 0) {
            // All of the old state is read before any of it is written.
            pack<T, V> last[H];
#pragma unroll
            for (int k = 0; k < H; ++k) {
                const int t = length - H + k;
                if (t >= 0) {
                    last[k] = load_pack<T, V>(x + t * s.x_stride);
                } else {
                    last[k] = in[0];
#pragma unroll
                    for (int m = 1; m < H; ++m)
                        if (length + k == m) last[k] = in[m];
                }
            }
            T* to = static_cast<T*>(a.state_out) + static_cast<long long>(slot) * H * s.channels + c.at;
#pragma unroll
            for (int k = 0; k < H; ++k)
                store_own<T, V>(to + static_cast<long long>(k) * s.channels, last[k], c.skip);
        }
        const auto outputs = [&](auto all) {
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                if (!decltype(all)::value && t0 + j >= s.n) break;
                pack<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float p = taps.bias[v];
#pragma unroll
                    for (int k = 0; k < K; ++k) p = fmaf(taps.w[k][v], to_float<T>(in[j + k][v]), p);
                    if constexpr (Silu) p *= opened(p);
                    out[v] = rounded<T>(decltype(all)::value || t0 + j < length ? p : 0.0f);
                }
                if (decltype(all)::value) store_pack<T, V>(y + j * s.y_stride, out);
                else store_own<T, V>(y + j * s.y_stride, out, c.skip);
            }
        };
        // The first tile's values may depend on states that another lane is replacing.
        if (whole && t0 + TS <= length && (c.skip == 0 || t0 > 0)) outputs(std::true_type{});
        else outputs(std::false_type{});
    }
}

// Steps of a lane backward, a multiple of kAhead; lanes of a workgroup along the channels; and the
// workgroups that share a channel.
struct ConvParts {
    int steps, across;
    int chunks;       // of a sequence, one a lane
    long long count;  // parts of the weights' gradients
};

constexpr int kAhead = 4;  // rows loaded at a time

// A lane takes a chunk of steps in blocks of kAhead rows, the next block's loads under way.  dxe of a
// step needs dp of the width - 1 steps behind it, so dx comes that many steps late, and a lane goes so
// many steps into the next chunk.  Blocks with all their steps in the chunk have no branches.
template <class T, int V, int K, bool Silu>
__global__ __launch_bounds__(kLanes) void conv_backward(ConvShape s, ConvBackward a, int vectors, ConvParts g) {
    constexpr int H = K - 1;
    __shared__ float lds[V * (K + 1)][kLanes];
    const int lane = threadIdx.x % g.across, row = threadIdx.x / g.across, rows = kLanes / g.across;
    const int slabs = (vectors + g.across - 1) / g.across;
    const long long part = blockIdx.x / slabs;
    const int vector = static_cast<int>(blockIdx.x - part * slabs) * g.across + lane;
    const long long chunk = part * rows + row;  // of all sequences
    const bool on = vector < vectors && chunk < static_cast<long long>(s.batch) * g.chunks;
    float dw[K][V] = {}, db[V] = {};
    const Channels c = channels_of<V>(min(vector, vectors - 1), s.channels);
    if (on) {
        const int b = static_cast<int>(chunk / g.chunks), t0 = static_cast<int>(chunk - static_cast<long long>(b) * g.chunks) * g.steps;
        const int length = length_of(a.lengths, b, s.n), t1 = min(t0 + g.steps, s.n);
        const long long first = b * static_cast<long long>(s.n);
        const T* x = static_cast<const T*>(a.x) + first * s.x_stride + c.at;
        const T* dy = static_cast<const T*>(a.dy) + first * s.y_stride + c.at;
        T* dx = static_cast<T*>(a.dx) + first * s.x_stride + c.at;
        const long long state = static_cast<long long>(b) * H * s.channels + c.at;
        const Taps<V, K> taps(a.weight, a.bias, c.at);
        // xe[j] and dp[j]: of the step H before the block's j-th.
        float xe[kAhead + H][V], dp[kAhead + H][V];
#pragma unroll
        for (int k = 0; k < H; ++k) {
            pack<T, V> in = {};
            if (t0 > 0) in = load_pack<T, V>(x + (t0 - H + k) * s.x_stride);
            else if (a.state_in) in = load_pack<T, V>(static_cast<const T*>(a.state_in) + state + static_cast<long long>(k) * s.channels);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                xe[kAhead + k][v] = t0 == 0 || t0 - H + k < length ? to_float<T>(in[v]) : 0.0f;
                dp[kAhead + k][v] = 0.0f;
            }
        }
        const int end = t1 + H;
        pack<T, V> nx[kAhead], ny[kAhead];
        const auto load = [&](int t) {
            if (t + kAhead <= s.n) {
                const T *from_x = x + t * s.x_stride, *from_y = dy + t * s.y_stride;
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    nx[j] = load_pack<T, V>(from_x + j * s.x_stride);
                    ny[j] = load_pack<T, V>(from_y + j * s.y_stride);
                }
            } else if (s.n > 0) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const long long at = min(t + j, s.n - 1);
                    nx[j] = load_pack<T, V>(x + at * s.x_stride);
                    ny[j] = load_pack<T, V>(dy + at * s.y_stride);
                }
            }
        };
        // Whole: every step counts, and so does each dx.
        const auto block = [&](auto whole, int t) {
            constexpr bool kWhole = decltype(whole)::value;
            pack<T, V> ys[kAhead];
#pragma unroll
            for (int k = 0; k < H; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    xe[k][v] = xe[kAhead + k][v];
                    dp[k][v] = dp[kAhead + k][v];
                }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                ys[j] = ny[j];
#pragma unroll
                for (int v = 0; v < V; ++v) xe[H + j][v] = kWhole || t + j < length ? to_float<T>(nx[j][v]) : 0.0f;
            }
            if (t + kAhead < end) load(t + kAhead);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int e = t + j;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float p = taps.bias[v];
#pragma unroll
                    for (int k = 0; k < K; ++k) p = fmaf(taps.w[k][v], xe[j + k][v], p);
                    float d = to_float<T>(ys[j][v]);
                    if constexpr (Silu) {
                        const float f = opened(p);
                        d *= fmaf(f * (1.0f - f), p, f);
                    }
                    d = kWhole || e < length ? d : 0.0f;
                    dp[H + j][v] = d;
                    if (kWhole || e < t1) {
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][v] = fmaf(d, xe[j + k][v], dw[k][v]);
                        db[v] += d;
                    }
                }
            }
            T* to = dx + (t - H) * s.x_stride;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int e = t + j;
                if (!kWhole && e >= end) break;
                pack<T, V> out, after = {};
                if (!kWhole && a.dstate_out && e >= length && e < length + H)
                    after = load_pack<T, V>(static_cast<const T*>(a.dstate_out) + state + static_cast<long long>(e - length) * s.channels);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float sum = kWhole ? 0.0f : to_float<T>(after[v]);
#pragma unroll
                    for (int k = 0; k < K; ++k) sum = fmaf(taps.w[k][v], dp[H + j - k][v], sum);
                    out[v] = rounded<T>(kWhole || e - H < length ? sum : 0.0f);
                }
                if (kWhole || e - H >= t0)
                    store_pack<T, V>(to + j * s.x_stride, out);
                else if (t0 == 0 && a.dstate_in)
                    store_pack<T, V>(static_cast<T*>(a.dstate_in) + state + static_cast<long long>(e) * s.channels, out);
            }
        };
        load(t0);
        for (int t = t0; t < end; t += kAhead) {
            if (t > t0 && t + kAhead <= t1 && t + kAhead <= length) block(std::true_type{}, t);
            else block(std::false_type{}, t);
        }
    }
    if (!a.dweight && !a.dbias) return;
    // The sums of the workgroup's rows, halving their number.
    for (int half = rows / 2; half > 0; half /= 2) {
        __syncthreads();
        if (row >= half && row < 2 * half) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int k = 0; k < K; ++k) lds[v * (K + 1) + k][threadIdx.x] = dw[k][v];
                lds[v * (K + 1) + K][threadIdx.x] = db[v];
            }
        }
        __syncthreads();
        if (row < half) {
            const int from = threadIdx.x + half * g.across;
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int k = 0; k < K; ++k) dw[k][v] += lds[v * (K + 1) + k][from];
                db[v] += lds[v * (K + 1) + K][from];
            }
        }
    }
    if (row == 0 && vector < vectors) {
        // workspace[part][tap, the last the bias][channel]
        float* to = a.workspace + part * (K + 1) * s.channels + c.at;
#pragma unroll
        for (int k = 0; k <= K; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v >= c.skip) to[static_cast<long long>(k) * s.channels + v] = k < K ? dw[k < K ? k : 0][v] : db[v];
    }
}

// Adds the parts of 32 sums: 32 lanes a sum, each every 32nd part.  Sums lie as [tap][channel].
__global__ __launch_bounds__(1024) void conv_add_parts(const float* parts, long long count, int channels, int width,
                                                       float* dweight, float* dbias) {
    __shared__ float lds[32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const long long sums = static_cast<long long>(width + 1) * channels;
    for (long long first = 32LL * blockIdx.x; first < sums; first += 32LL * gridDim.x) {
        float sum = 0.0f;
        if (first + lane < sums) {
#pragma unroll 4
            for (long long k = group; k < count; k += 32) sum += parts[k * sums + first + lane];
        }
        __syncthreads();
        lds[group][lane] = sum;
        __syncthreads();
        sum = lds[lane][group];
#pragma unroll
        for (int m = 1; m < 32; m *= 2) sum += __shfl_xor(sum, m);
        const long long at = first + group;
        if (lane == 0 && at < sums) {
            const long long tap = at / channels, c = at - tap * channels;
            if (tap < width) {
                if (dweight) dweight[c * width + tap] = sum;
            } else if (dbias) {
                dbias[c] = sum;
            }
        }
    }
}

template <class F>
auto with_type(int precision, F f) {
    if (precision == THFF_FLOAT) return f(float{});
    if (precision == THFF_HALF) return f(half_t{});
    return f(bfloat_t{});
}

template <int V_, int K_>
struct Kind {
    static constexpr int V = V_, K = K_;
};

// V channels a lane; fewer channels than that, one.
template <int V, class F>
auto with_kind(const ConvShape& s, F f) {
    if (s.channels < V) {
        if (s.width == 2) return f(Kind<1, 2>{});
        if (s.width == 3) return f(Kind<1, 3>{});
        return f(Kind<1, 4>{});
    }
    if (s.width == 2) return f(Kind<V, 2>{});
    if (s.width == 3) return f(Kind<V, 3>{});
    return f(Kind<V, 4>{});
}

// Backward, where a channel takes four times the registers: 4 channels a lane from 2^25 values on, for
// whole sectors of rows that lie apart, and 2 of fewer, for more lanes.  us of both passes by 4 and 2,
// bfloat16: 8 x 4096 x 2048 in a projection's rows 124 and 139 (8, backward alone: 143 for 75), 1 x
// 65536 x 1024 137 and 141; 16 x 2048 x 768 63.5 and 61.2, 2 x 2048 x 1024 23.2 and 21.6; float 8 x
// 4096 x 2048 in a projection's rows 230 and 251, 4 x 2048 x 1024 45 and 35.
template <class F>
auto with_backward_kind(const ConvShape& s, F f) {
    const __int128 values = static_cast<__int128>(s.batch) * s.n * s.channels;
    return values < 1 << 25 ? with_kind<2>(s, f) : with_kind<4>(s, f);
}

int vectors_of(const ConvShape& s, int v) { return (s.channels + v - 1) / v; }

ConvParts parts_of(const ConvShape& s, int v) {
    // Lanes, and the least steps of one, which goes width - 1 steps on into the next's: twice the lanes
    // take 128 us for 124 at bfloat16 8 x 4096 x 2048, at 2 x 2048 x 1024 32 steps 22.7 and 8 steps 21.7
    // for 21.6.
    constexpr long long kWanted = 1 << 17, kLeast = 16;
    ConvParts g;
    const int vectors = vectors_of(s, v);
    g.across = 1;
    while (g.across < 64 && g.across < vectors) g.across *= 2;
    const long long steps = static_cast<long long>(s.batch) * s.n * vectors / kWanted;
    g.steps = static_cast<int>(std::min<long long>(std::max(steps, kLeast), 1 << 20)) / kAhead * kAhead;
    g.chunks = std::max(1, static_cast<int>((s.n + static_cast<long long>(g.steps) - 1) / g.steps));
    const int rows = kLanes / g.across;
    g.count = (static_cast<long long>(s.batch) * g.chunks + rows - 1) / rows;
    return g;
}

template <class T, int V, int K, bool Silu, int TS>
hipError_t launch_forward(const ConvShape& s, const ConvForward& a, hipStream_t stream) {
    const int vectors = vectors_of(s, V);
    const long long tiles = std::max<long long>(1, (s.n + TS - 1LL) / TS);
    const __int128 lanes = static_cast<__int128>(s.batch) * tiles * vectors;
    const long long blocks = static_cast<long long>(std::min<__int128>((lanes + kLanes - 1) / kLanes, 1 << 23));
    conv_forward<T, V, K, Silu, TS><<<static_cast<unsigned>(blocks), kLanes, 0, stream>>>(s, a, vectors, tiles);
    return hipGetLastError();
}

}  // namespace

long long conv_workspace_bytes(const ConvShape& s) {
    if (s.batch == 0 || s.n == 0 || s.channels == 0) return 0;
    const long long parts = with_type(s.precision, [&](auto v) {
        return with_backward_kind(s, [&](auto kind) { return parts_of(s, decltype(kind)::V).count; });
    });
    return 4 * parts * (s.width + 1) * s.channels;
}

hipError_t launch_short_conv(const ConvShape& s, const ConvForward& a, hipStream_t stream) {
    return with_type(s.precision, [&](auto v) {
        using T = decltype(v);
        return with_kind<16 / sizeof(T)>(s, [&](auto kind) {
            using Q = decltype(kind);
            if (s.n <= 1)
                return s.silu ? launch_forward<T, Q::V, Q::K, true, 1>(s, a, stream)
                              : launch_forward<T, Q::V, Q::K, false, 1>(s, a, stream);
            return s.silu ? launch_forward<T, Q::V, Q::K, true, kSteps>(s, a, stream)
                          : launch_forward<T, Q::V, Q::K, false, kSteps>(s, a, stream);
        });
    });
}

hipError_t launch_short_conv_backward(const ConvShape& s, const ConvBackward& a, hipStream_t stream) {
    return with_type(s.precision, [&](auto v) {
        using T = decltype(v);
        return with_backward_kind(s, [&](auto kind) {
            using Q = decltype(kind);
            const int vectors = vectors_of(s, Q::V);
            const ConvParts g = parts_of(s, Q::V);
            const bool none = s.batch == 0 || s.n == 0;
            ConvBackward call = a;
            if (none) call.dweight = call.dbias = nullptr;
            if (s.batch > 0) {
                const long long slabs = (vectors + g.across - 1) / g.across;
                const auto kernel = s.silu ? conv_backward<T, Q::V, Q::K, true> : conv_backward<T, Q::V, Q::K, false>;
                kernel<<<static_cast<unsigned>(g.count * slabs), kLanes, 0, stream>>>(s, call, vectors, g);
            }
            if (a.dweight || a.dbias) {
                const long long sums = static_cast<long long>(s.width + 1) * s.channels;
                conv_add_parts<<<static_cast<unsigned>(std::min<long long>((sums + 31) / 32, 1 << 20)), 1024, 0, stream>>>(
                    a.workspace, none ? 0 : g.count, s.channels, s.width, a.dweight, a.dbias);
            }
            return hipGetLastError();
        });
    });
}

}  // namespace thff
