// scan.hip -- the gated linear recurrence: per channel, with f = sigmoid(gate),
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  y[t] = h[t],
// and its gradients: lam[t] = dy[t] + f[t+1] lam[t+1],
//   dx[t] = (1 - f[t]) lam[t],  dgate[t] = lam[t] (h[t-1] - x[t]) f[t] (1 - f[t]).
// Values of steps at or past a sequence's length reach no result.
#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {
namespace {

// Steps between the states that the forward pass saves for the backward pass.
constexpr int kSavedSteps = 16;
constexpr int kLanes = 256;

struct Gate {
    float keep;   // sigmoid(g)
    float enter;  // 1 - sigmoid(g) = sigmoid(-g)
};

// Both from e = exp(-|g|) <= 1, so that neither overflows nor cancels.
__device__ __forceinline__ Gate gate_of(float g) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(g));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    const float s = e * r;
    return g >= 0.0f ? Gate{r, s} : Gate{s, r};
}

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

__device__ __forceinline__ int length_of(const int* lengths, int b, int n) {
    return lengths ? min(max(lengths[b], 0), n) : n;
}

// Row of the state pool for sequence b, or -1 (none).
__device__ __forceinline__ int state_row(const ScanShape& s, const int* slots, int b) {
    if (!slots) return b;
    const int row = slots[b];
    return row >= 0 && row < s.states ? row : -1;
}

template <class T>
__global__ __launch_bounds__(kLanes) void scan_forward(ScanShape s, ScanForward a) {
    const long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x;
    if (i >= static_cast<long long>(s.batch) * s.channels) return;
    const int b = static_cast<int>(i / s.channels), c = static_cast<int>(i % s.channels);
    const int len = length_of(a.lengths, b, s.n), row = state_row(s, a.slots, b);
    const long long state = static_cast<long long>(row) * s.channels + c;
    const int chunks = (s.n + kSavedSteps - 1) / kSavedSteps;
    Element e = first_element(s, b, c);
    float h = a.state_in && row >= 0 ? a.state_in[state] : 0.0f;
    for (int t = 0; t < s.n; ++t) {
        if (a.saved && t % kSavedSteps == 0)
            a.saved[(static_cast<long long>(b) * chunks + t / kSavedSteps) * s.channels + c] = h;
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
    const int chunks = (s.n + kSavedSteps - 1) / kSavedSteps;
    const Element e = first_element(s, b, c);
    const T* x = static_cast<const T*>(a.x) + e.x;
    const T* gate = static_cast<const T*>(a.gate) + e.gate;
    const T* dy = static_cast<const T*>(a.dy) + e.y;
    T* dx = static_cast<T*>(a.dx) + e.x;
    T* dgate = static_cast<T*>(a.dgate) + e.gate;
    float carried = a.dstate_out ? a.dstate_out[i] : 0.0f;
    for (int chunk = chunks - 1; chunk >= 0; --chunk) {
        const int t0 = chunk * kSavedSteps;
        float before[kSavedSteps];
        float h = a.saved[(static_cast<long long>(b) * chunks + chunk) * s.channels + c];
        for (int k = 0; k < kSavedSteps; ++k) {
            before[k] = h;
            if (t0 + k < len) {
                const Gate g = gate_of(to_float(gate[(t0 + k) * e.gate_step]));
                h = fmaf(g.keep, h, g.enter * to_float(x[(t0 + k) * e.x_step]));
            }
        }
        for (int k = kSavedSteps - 1; k >= 0; --k) {
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

}  // namespace

long long scan_saved_bytes(const ScanShape& s) {
    const long long chunks = (static_cast<long long>(s.n) + kSavedSteps - 1) / kSavedSteps;
    return 4 * chunks * s.batch * s.channels;
}

long long scan_workspace_bytes(const ScanShape&) { return 0; }

bool scan_fits(const ScanShape& s) {
    return static_cast<long long>(s.batch) * s.channels <= 0x7fffffffLL;
}

hipError_t launch_gated_scan(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    const unsigned blocks = blocks_of(s);
    if (s.precision == THFF_FLOAT)
        scan_forward<float><<<blocks, kLanes, 0, stream>>>(s, a);
    else if (s.precision == THFF_HALF)
        scan_forward<half_t><<<blocks, kLanes, 0, stream>>>(s, a);
    else
        scan_forward<bfloat_t><<<blocks, kLanes, 0, stream>>>(s, a);
    return hipGetLastError();
}

hipError_t launch_gated_scan_backward(const ScanShape& s, const ScanBackward& a,
                                      hipStream_t stream) {
    const unsigned blocks = blocks_of(s);
    if (s.precision == THFF_FLOAT)
        scan_backward<float><<<blocks, kLanes, 0, stream>>>(s, a);
    else if (s.precision == THFF_HALF)
        scan_backward<half_t><<<blocks, kLanes, 0, stream>>>(s, a);
    else
        scan_backward<bfloat_t><<<blocks, kLanes, 0, stream>>>(s, a);
    return hipGetLastError();
}

}  // namespace thff
