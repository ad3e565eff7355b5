// scan.hip -- the gated linear recurrence: per channel, with f = sigmoid(gate),
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  y[t] = h[t],
// and its gradients: lam[t] = dy[t] + f[t+1] lam[t+1],
//   dx[t] = (1 - f[t]) lam[t],  dgate[t] = lam[t] (h[t-1] - x[t]) f[t] (1 - f[t]).
// Values of steps at or past a sequence's length reach no result.
#include <algorithm>

#include "scan_last.hpp"
#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {
namespace {

// Steps between the saved states of the channels-first kernels.
constexpr int kChunk = 16;
constexpr int kLanes = 256;

struct Element {
    long long x, gate, y;  // offsets of step t
    long long x_step, gate_step, y_step;
};

__device__ __forceinline__ Element first_element(const ScanShape& s, int b, int c) {
    if (s.channels_first) {
        const long long row = static_cast<long long>(b) * s.channels + c;
        return {row * s.x_stride, row * s.gate_stride, row * s.y_stride, 1, 1, 1};
    }
    const long long row = static_cast<long long>(b) * s.n;
    return {row * s.x_stride + c, row * s.gate_stride + c, row * s.y_stride + c,
            s.x_stride, s.gate_stride, s.y_stride};
}

template <class T>
__global__ __launch_bounds__(kLanes) void scan_forward(ScanShape s, ScanForward a) {
    const long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x;
    if (i >= static_cast<long long>(s.batch) * s.channels) return;
    const int b = static_cast<int>(i / s.channels), c = static_cast<int>(i % s.channels);
    const int len = length_of(a.lengths, b, s.n), row = state_row(s, a.slots, b);
    const long long state = static_cast<long long>(row) * s.channels + c;
    const int chunks = (s.n + kChunk - 1) / kChunk;
    Element e = first_element(s, b, c);
    float h = a.state_in && row >= 0 ? a.state_in[state] : 0.0f;
    for (int t = 0; t < s.n; ++t) {
        if (a.saved && t % kChunk == 0)
            a.saved[(static_cast<long long>(b) * chunks + t / kChunk) * s.channels + c] = h;
        float out = 0.0f;
        if (t < len) {
            const Gate g = gate_of(to_float(static_cast<const T*>(a.gate)[e.gate]));
            h = fmaf(g.keep, h, g.enter * to_float(static_cast<const T*>(a.x)[e.x]));
            out = h;
        }
        static_cast<T*>(a.y)[e.y] = from_float<T>(out);
        e.x += e.x_step, e.gate += e.gate_step, e.y += e.y_step;
    }
    if (a.state_out && row >= 0) a.state_out[state] = h;
}

template <class T>
__global__ __launch_bounds__(kLanes) void scan_backward(ScanShape s, ScanBackward a) {
    const long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x;
    if (i >= static_cast<long long>(s.batch) * s.channels) return;
    const int b = static_cast<int>(i / s.channels), c = static_cast<int>(i % s.channels);
    const int len = length_of(a.lengths, b, s.n);
    const int chunks = (s.n + kChunk - 1) / kChunk;
    const Element e = first_element(s, b, c);
    const T* x = static_cast<const T*>(a.x) + e.x;
    const T* gate = static_cast<const T*>(a.gate) + e.gate;
    const T* dy = static_cast<const T*>(a.dy) + e.y;
    T* dx = static_cast<T*>(a.dx) + e.x;
    T* dgate = static_cast<T*>(a.dgate) + e.gate;
    float carried = a.dstate_out ? a.dstate_out[i] : 0.0f;
    for (int chunk = chunks - 1; chunk >= 0; --chunk) {
        const int t0 = chunk * kChunk;
        float before[kChunk];
        float h = a.saved[(static_cast<long long>(b) * chunks + chunk) * s.channels + c];
        for (int k = 0; k < kChunk; ++k) {
            before[k] = h;
            if (t0 + k < len) {
                const Gate g = gate_of(to_float(gate[(t0 + k) * e.gate_step]));
                h = fmaf(g.keep, h, g.enter * to_float(x[(t0 + k) * e.x_step]));
            }
        }
        for (int k = kChunk - 1; k >= 0; --k) {
            const int t = t0 + k;
            if (t >= s.n) continue;
            float gx = 0.0f, gg = 0.0f;
            if (t < len) {
                const Gate g = gate_of(to_float(gate[t * e.gate_step]));
                const float lam = to_float(dy[t * e.y_step]) + carried;
                gx = g.enter * lam;
                gg = lam * (before[k] - to_float(x[t * e.x_step])) * g.keep * g.enter;
                carried = g.keep * lam;
            }
            dx[t * e.x_step] = from_float<T>(gx);
            dgate[t * e.gate_step] = from_float<T>(gg);
        }
    }
    if (a.dstate_in) a.dstate_in[i] = carried;
}

unsigned blocks_of(const ScanShape& s) {
    return static_cast<unsigned>((static_cast<long long>(s.batch) * s.channels + kLanes - 1) /
                                 kLanes);
}

// Sets the counters of a chain to zero and empties its words.  (A kernel: a captured memset
// is not replayed reliably.)
__global__ __launch_bounds__(kLanes) void clear_chain(uint4* to, long long counters,
                                                      long long count) {
    const long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x;
    if (i >= count) return;
    const unsigned v = i < counters ? 0u : ~0u;
    to[i] = make_uint4(v, v, v, v);
}

// Calls f with the tile type of a shape's forward or backward pass: 4 bytes a lane and row;
// lanes along the channels all 64 of a wave, or 16 where that leaves far fewer of them idle.
template <class T, bool Backward, class F>
auto with_tile(const ScanShape& s, F f) {
    constexpr int VEC = 4 / sizeof(T);
    using Wide = std::conditional_t<Backward, Tile<VEC, 64, 8, 14, 2, 4>, Tile<VEC, 64, 8, 14, 2, 8>>;
    using Thin = std::conditional_t<Backward, Tile<VEC, 16, 8, 14, 2, 4>, Tile<VEC, 16, 8, 14, 2, 8>>;
    const auto taken = [&](long long channels) {
        return (s.channels + channels - 1) / channels * channels;
    };
    const bool thin = 4 * taken(Wide::kChannels) > 5 * taken(Thin::kChannels);
    return thin ? f(Thin{}) : f(Wide{});
}

// Calls f with a value of the shape's type.
template <class F>
auto with_type(const ScanShape& s, F f) {
    if (s.precision == THFF_FLOAT) return f(float{});
    if (s.precision == THFF_HALF) return f(half_t{});
    return f(bfloat_t{});
}

template <class L>
Chain chain_of(const ScanShape& s, void* workspace) {
    Chain chain;
    chain.slabs = (s.channels + L::kChannels - 1) / L::kChannels;
    chain.tiles = s.n > 0 ? (s.n + L::kSteps - 1) / L::kSteps : 1;
    chain.columns = static_cast<unsigned>(s.batch) * chain.slabs;
    chain.drawn = static_cast<unsigned*>(workspace);
    chain.words = reinterpret_cast<Word*>(static_cast<char*>(workspace) +
                                          static_cast<long long>(chain.columns) * kCounterBytes);
    return chain;
}

template <class L>
long long chain_bytes(const ScanShape& s) {
    const Chain chain = chain_of<L>(s, nullptr);
    if (chain.tiles <= 1) return 0;
    return chain.columns * (kCounterBytes + 8LL * L::kChannels * chain.tiles);
}

template <class L>
bool chain_fits(const ScanShape& s) {
    const Chain chain = chain_of<L>(s, nullptr);
    return static_cast<__int128>(s.batch) * chain.slabs * chain.tiles <= 0x7fffffff;
}

template <class T, class L, class Args>
hipError_t launch_last(void (*kernel)(ScanShape, Args, Chain), const ScanShape& s, const Args& a,
                       hipStream_t stream) {
    const Chain chain = chain_of<L>(s, a.workspace);
    const long long bytes = chain_bytes<L>(s);
    if (bytes) {
        const long long count = bytes / 16;
        clear_chain<<<static_cast<unsigned>((count + kLanes - 1) / kLanes), kLanes, 0, stream>>>(
            static_cast<uint4*>(a.workspace), chain.columns * (kCounterBytes / 16LL), count);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    kernel<<<chain.columns * chain.tiles, L::kLanes, 0, stream>>>(s, a, chain);
    return hipGetLastError();
}

}  // namespace

long long scan_saved_bytes(const ScanShape& s) {
    const int steps = s.channels_first ? kChunk : kSaved;
    const long long chunks = (static_cast<long long>(s.n) + steps - 1) / steps;
    return 4 * chunks * s.batch * s.channels;
}

long long scan_workspace_bytes(const ScanShape& s) {
    if (s.channels_first) return 0;
    const auto bytes = [&](auto tile) { return chain_bytes<decltype(tile)>(s); };
    return with_type(s, [&](auto v) {
        using T = decltype(v);
        return std::max(with_tile<T, false>(s, bytes), with_tile<T, true>(s, bytes));
    });
}

bool scan_fits(const ScanShape& s) {
    if (static_cast<long long>(s.batch) * s.channels > 0x7fffffffLL) return false;
    if (s.channels_first) return true;
    const auto fits = [&](auto tile) { return chain_fits<decltype(tile)>(s); };
    return with_type(s, [&](auto v) {
        using T = decltype(v);
        return with_tile<T, false>(s, fits) && with_tile<T, true>(s, fits);
    });
}

template <class T>
hipError_t forward_of(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    if (s.channels_first) {
        scan_forward<T><<<blocks_of(s), kLanes, 0, stream>>>(s, a);
        return hipGetLastError();
    }
    return with_tile<T, false>(s, [&](auto tile) {
        using L = decltype(tile);
        return launch_last<T, L>(scan_last_forward<T, L>, s, a, stream);
    });
}

template <class T>
hipError_t backward_of(const ScanShape& s, const ScanBackward& a, hipStream_t stream) {
    if (s.channels_first) {
        scan_backward<T><<<blocks_of(s), kLanes, 0, stream>>>(s, a);
        return hipGetLastError();
    }
    return with_tile<T, true>(s, [&](auto tile) {
        using L = decltype(tile);
        return launch_last<T, L>(scan_last_backward<T, L>, s, a, stream);
    });
}

hipError_t launch_gated_scan(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    return with_type(s, [&](auto v) { return forward_of<decltype(v)>(s, a, stream); });
}

hipError_t launch_gated_scan_backward(const ScanShape& s, const ScanBackward& a,
                                      hipStream_t stream) {
    return with_type(s, [&](auto v) { return backward_of<decltype(v)>(s, a, stream); });
}

}  // namespace thff
