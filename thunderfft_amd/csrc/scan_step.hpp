// scan_step.hpp -- one step of the gated recurrence (n = 1: a token of each sequence): no
// tiles, no chain; a lane takes V channels of a sequence.  Latency bounds it: bfloat16 8 x 1024
// takes 3.1 us, half 256 x 4096 4.7 us (14.7 MB, 3.1 TB/s, most of it from the caches).
#pragma once

#include "scan_chain.hpp"

namespace thff {

constexpr int kStepLanes = 256;

// Elements between the values of a sequence's neighbouring channels, and of its first to the
// next sequence's: both layouts are one for a single step.
struct StepStrides {
    long long x, gate, y;
    long long x_row, gate_row, y_row;
};

// Vectors where V > 1 (neighbouring channels lie side by side); the last lane of a sequence may
// have fewer channels.
template <class T, int V>
__global__ __launch_bounds__(kStepLanes) void scan_step(ScanShape s, ScanForward a, StepStrides d) {
    const int lanes = (s.channels + V - 1) / V;
    const long long i = static_cast<long long>(blockIdx.x) * kStepLanes + threadIdx.x;
    const int b = static_cast<int>(i / lanes);
    if (b >= s.batch) return;
    const int c = static_cast<int>(i - static_cast<long long>(b) * lanes) * V;
    const int some = min(V, s.channels - c), row = state_row(s, a.slots, b);
    const bool on = length_of(a.lengths, b, 1) > 0;
    const long long at = static_cast<long long>(row) * s.channels + c;
    const T* x = static_cast<const T*>(a.x) + b * d.x_row + c * d.x;
    const T* gate = static_cast<const T*>(a.gate) + b * d.gate_row + c * d.gate;
    T* y = static_cast<T*>(a.y) + b * d.y_row + c * d.y;
    const bool stored = a.state_in && row >= 0;
    pack<float, V> h = {};
    pack<T, V> in = {}, g = {}, out;
    if (some == V) {
        in = load_pack<T, V>(x);
        g = load_pack<T, V>(gate);
        if (stored) h = load_pack<float, V>(a.state_in + at);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < some) {
                in[v] = x[v];
                g[v] = gate[v];
                if (stored) h[v] = a.state_in[at + v];
            }
    }
    if (a.saved) {
        const long long to = static_cast<long long>(b) * s.channels + c;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < some) a.saved[to + v] = h[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Gate q = gate_of(to_float<T>(g[v]));
        const float next = fmaf(q.keep, h[v], q.enter * to_float<T>(in[v]));
        if (on) h[v] = next;
        out[v] = from_float<T>(on ? next : 0.0f);
    }
    store_some<T, V>(y, out, some);
    if (a.state_out && row >= 0) {
        // Through the caches: the next token reads it soon.
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < some) a.state_out[at + v] = h[v];
    }
}

}  // namespace thff
