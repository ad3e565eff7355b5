// state_scan.hip -- the state space scan: for each channel and each of its states,
//   dt = log(1 + exp(delta + delta_bias)),  h[t] = exp(dt a) h[t-1] + dt x[t] b[t],
//   y[t] = (sum over the states of c[t] h[t] + skip x[t]) gate[t] / (1 + exp(-gate[t])),
// and its gradients; how it is cut into workgroups.  The kernels are in state_kernels.hpp.
#include <algorithm>

#include "sequence_io.hpp"
#include "state_cut.hpp"

namespace thff {
namespace {

Cut cut_of(const StateShape& s) {
    return with_lanes(s.order, [&](auto lanes) {
        using L = decltype(lanes);
        Cut cut;
        const int each = s.channels / s.groups;
        cut.padded = L::P;
        cut.slabs = (each + L::kSlab - 1) / L::kSlab;
        cut.segments = 1;
        cut.steps = (s.n + kStateBlock - 1) / kStateBlock * kStateBlock;
        cut.blocks = static_cast<long long>(s.batch) * s.groups * cut.slabs * cut.segments;
        return cut;
    });
}

template <class F>
auto with_type(int precision, F f) {
    if (precision == THFF_FLOAT) return f(float{});
    if (precision == THFF_HALF) return f(half_t{});
    return f(bfloat_t{});
}

}  // namespace

long long state_saved_bytes(const StateShape& s) {
    const long long tiles = (s.n + kStateTile - 1) / kStateTile;
    return 4 * s.batch * tiles * s.channels * cut_of(s).padded;
}

long long state_workspace_bytes(const StateShape& s) {
    if (s.channels == 0) return 0;
    return Parts(s, cut_of(s)).bytes(s);
}

bool state_fits(const StateShape& s) {
    const Cut cut = cut_of(s);
    // Sizes of the buffers in bytes, from above.
    const __int128 rows = static_cast<__int128>(s.batch) * s.n;
    const __int128 shared = rows * s.groups * cut.slabs * 2 * cut.padded;
    const __int128 states = (static_cast<__int128>(s.batch) * cut.segments + rows / kStateTile + s.batch) * s.channels * (cut.padded + 4);
    return 4 * (shared + 2 * states) < static_cast<__int128>(1) << 62 && cut.blocks <= 1LL << 36;
}

hipError_t launch_state_scan(const StateShape& s, const StateForward& a, hipStream_t stream) {
    const Cut cut = cut_of(s);
    return with_type(s.precision, [&](auto v) { return launch_state_forward<decltype(v)>(s, a, cut, stream); });
}

hipError_t launch_state_scan_backward(const StateShape& s, const StateBackward& a, hipStream_t stream) {
    const Cut cut = cut_of(s);
    return with_type(s.precision, [&](auto v) { return launch_state_backward<decltype(v)>(s, a, cut, stream); });
}

}  // namespace thff
