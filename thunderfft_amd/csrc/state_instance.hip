// state_instance.hip -- the state space scan for one type of values, THFF_STATE_TYPE.
#include "state_kernels.hpp"

namespace thff {
namespace {

dim3 grid_of(long long blocks) {
    // A launch has less than 2^32 lanes along x, so many workgroups take rows of a grid.
    constexpr long long kMost = 1LL << 21;
    return dim3(static_cast<unsigned>(std::min(blocks, kMost)), static_cast<unsigned>((blocks + kMost - 1) / kMost));
}

// From so many lanes on a lane of a single step takes two sequences: half 256 x 4096 of 16 states 23 us
// against 27 by one (and 29 by four), 128 x 4096 14 against 16, 32 x 4096 9 to 10 us a call by either;
// with less lanes half as many do not fill the card.
constexpr long long kManyLanes = 1 << 20;

// Lanes of a channel for one step.
template <class F>
auto with_step_lanes(int order, F f) {
    if (order <= 4) return f(std::integral_constant<int, 1>{});
    if (order <= 8) return f(std::integral_constant<int, 2>{});
    if (order <= 16) return f(std::integral_constant<int, 4>{});
    if (order <= 32) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{});
}

}  // namespace

template <class T>
hipError_t launch_state_forward(const StateShape& s, const StateForward& a, const Cut& cut, hipStream_t stream) {
    // A single step that saves nothing.
    if (s.n == 1 && !a.saved)
        return with_step_lanes(s.order, [&](auto lanes) {
            constexpr int N = decltype(lanes)::value;
            const auto launch = [&](auto kernel, int rows) {
                const long long count = static_cast<long long>((s.batch + rows - 1) / rows) * s.channels * N;
                kernel<<<grid_of((count + kLanes - 1) / kLanes), kLanes, 0, stream>>>(s, a);
                return hipGetLastError();
            };
            return static_cast<long long>(s.batch) * s.channels * N < kManyLanes ? launch(state_step<T, N, 1>, 1)
                                                                                : launch(state_step<T, N, 2>, 2);
        });
    return with_forward_lanes(s, [&](auto lanes) {
        using L = decltype(lanes);
        const auto launch = [&](auto kernel) {
            kernel<<<grid_of(cut.blocks), L::kLanes, 0, stream>>>(s, a, cut);
            return hipGetLastError();
        };
        if (cut.segments > 1) {
            const hipError_t err = launch(state_forward<T, L, true, false, false>);
            if (err != hipSuccess) return err;
        }
        if (a.saved) return a.gate ? launch(state_forward<T, L, false, true, true>) : launch(state_forward<T, L, false, true, false>);
        return a.gate ? launch(state_forward<T, L, false, false, true>) : launch(state_forward<T, L, false, false, false>);
    });
}

template <class T>
hipError_t launch_state_backward(const StateShape& s, const StateBackward& a, const Cut& cut, hipStream_t stream) {
    return with_lanes(s.order, [&](auto lanes) {
        using L = decltype(lanes);
        if (s.batch > 0) {
            if (cut.segments > 1) {
                state_backward<T, L, true><<<grid_of(cut.blocks), L::kLanes, 0, stream>>>(s, a, cut);
                const hipError_t err = hipGetLastError();
                if (err != hipSuccess) return err;
            }
            state_backward<T, L, false><<<grid_of(cut.blocks), L::kLanes, 0, stream>>>(s, a, cut);
            const hipError_t err = hipGetLastError();
            if (err != hipSuccess) return err;
        }
        const long long sums = static_cast<long long>(s.channels) * (cut.padded + 2);
        const long long shared = static_cast<long long>(s.batch) * s.n * s.groups * 2 * cut.padded / 4;
        const int few = static_cast<int>(std::min((sums + 31) / 32, 1LL << 20));
        const long long many = std::min((shared + kLanes - 1) / kLanes, 1LL << 20);
        add_state_parts<T><<<static_cast<unsigned>(few + many), kLanes, 0, stream>>>(s, a, cut, few);
        return hipGetLastError();
    });
}

template hipError_t launch_state_forward<THFF_STATE_TYPE>(const StateShape&, const StateForward&, const Cut&,
                                                          hipStream_t);
template hipError_t launch_state_backward<THFF_STATE_TYPE>(const StateShape&, const StateBackward&, const Cut&,
                                                           hipStream_t);

}  // namespace thff
