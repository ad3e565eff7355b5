// state_scan.hip -- the state space scan: for each channel and each of its states,
//   dt = log(1 + exp(delta + delta_bias)),  h[t] = exp(dt a) h[t-1] + dt x[t] b[t],
//   y[t] = (sum over the states of c[t] h[t] + skip x[t]) gate[t] / (1 + exp(-gate[t])),
// and its gradients; how it is cut into workgroups.  The kernels are in state_kernels.hpp.
#include <algorithm>

#include "sequence_io.hpp"
#include "state_cut.hpp"

namespace thff {
namespace {

// Segments of the steps.  They cost a kernel over the steps that only finds the segments' ends, 0.7
// (forward) and 0.24 (backward) of the time of the steps themselves, and where there is one wave a
// SIMD (1024 in all) the steps take 0.8 of it with two and more.  Order 16, us a call by one segment
// against many: forward bfloat16 6 x 4096 x 2048 (1536 waves of 8 lanes) 367 against 410, 8 x 4096 x
// 2048 (1024 of 4) 390 against 490, 1 x 256 x 2048 (128) 27 against 20, 1 x 65536 x 1024 (64) 5316
// against 469; backward 8 x 4096 x 2048 1224 against 1106, float 33 x 512 x 96 in two groups (264)
// 174 against 67.
//
// A segment goes through the ends of all before it, so that their number should be small against
// their steps: not more of them than steps in each up to 2 waves a SIMD, and 1/16 of the steps beyond,
// up to 4.  bfloat16, forward + backward, against 4 waves a SIMD whatever the steps: 1 x 65536 x 64
// (256 segments for 1024) 145 + 249 us against 490 + 549, 1 x 16384 x 512 (64 for 128) 99 + 177
// against 126 + 213, 4 x 1024 x 1024 (8 for 16) 48 + 92 against 56 + 101.  8 waves a SIMD are no
// faster backward: 8 x 4096 x 2048 1103 us against 1085, 2 x 4096 x 1024 210 against 167.
//
// All of it at order 16, 4 states a lane.  Waves of lower orders have less work a step, and the thresholds,
// which count waves, have not been measured there.
int segments_of(long long waves, int n, bool backward) {
    if (waves == 0 || waves > (backward ? 1024 : 832) || n < (backward ? 128 : 256)) return 1;
    int segments = 1;
    while (segments < n / 64 && segments * waves < 4096) {
        const long long more = segments + 1;
        if (more * more * (segments * waves < 2048 ? 1 : 16) > n) break;
        ++segments;
    }
    return segments;
}

template <class L>
Cut cut_with(const StateShape& s, bool backward) {
    Cut cut;
    cut.padded = L::P;
    cut.slabs = slabs_of<L>(s);
    const int blocks = (s.n + kStateBlock - 1) / kStateBlock;
    const int want = segments_of(waves_of<L>(s), s.n, backward);
    cut.steps = (blocks + want - 1) / want * kStateBlock;
    cut.segments = s.n > 0 ? (s.n + cut.steps - 1) / cut.steps : 1;
    cut.blocks = static_cast<long long>(s.batch) * s.groups * cut.slabs * cut.segments;
    return cut;
}

Cut cut_of(const StateShape& s, bool backward) {
    const auto cut = [&](auto lanes) { return cut_with<decltype(lanes)>(s, backward); };
    return backward ? with_lanes(s.order, cut) : with_forward_lanes(s, cut);
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
    return 4LL * s.batch * tiles * s.channels * cut_of(s, false).padded;
}

long long state_forward_bytes(const StateShape& s) {
    return s.channels == 0 ? 0 : 4 * Parts(s, cut_of(s, false)).shared;
}

long long state_workspace_bytes(const StateShape& s) {
    return s.channels == 0 ? 0 : std::max(state_forward_bytes(s), Parts(s, cut_of(s, true)).bytes(s));
}

bool state_fits(const StateShape& s) {
    // Sizes of the buffers in bytes, from above.
    const Cut cut = cut_of(s, true);
    const __int128 rows = static_cast<__int128>(s.batch) * s.n;
    const __int128 shared = rows * s.groups * cut.slabs * 2 * cut.padded;
    const __int128 states = (static_cast<__int128>(s.batch) * (cut.segments + 1) + rows / kStateTile) * s.channels * (cut.padded + 4);
    return 4 * (shared + 2 * states) < static_cast<__int128>(1) << 62 && cut.blocks <= 1LL << 36;
}

hipError_t launch_state_scan(const StateShape& s, const StateForward& a, hipStream_t stream) {
    const Cut cut = cut_of(s, false);
    return with_type(s.precision, [&](auto v) { return launch_state_forward<decltype(v)>(s, a, cut, stream); });
}

hipError_t launch_state_scan_backward(const StateShape& s, const StateBackward& a, hipStream_t stream) {
    const Cut cut = cut_of(s, true);
    return with_type(s.precision, [&](auto v) { return launch_state_backward<decltype(v)>(s, a, cut, stream); });
}

}  // namespace thff
