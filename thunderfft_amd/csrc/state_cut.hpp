// state_cut.hpp -- how the state space scan is cut into workgroups, and what its translation units
// (state_instance.hip, one for each type of values) offer.
#pragma once

#include "block.hpp"

namespace thff {

constexpr int kStateBlock = 32;  // steps whose b and c are in LDS at a time, forward
constexpr long long kStateStride = 1 << 24;  // the longest: offsets of a lane's rows fit 32 bits
constexpr int kStateTile = 16;   // steps between saved states, and of the backward pass at a time

// S states of a channel on each of LPC neighbouring lanes, in workgroups of W waves.  4 lanes a channel
// are as few as let each load whole sectors and share the work that is once a step; 8 waves a
// workgroup leave half of the compute units without one where channels are few.
template <int S_, int LPC_, int W_>
struct Lanes {
    static constexpr int S = S_, LPC = LPC_, W = W_, P = S * LPC, kLanes = 64 * W, kWave = 64 / LPC, kSlab = W * kWave;
};

// Calls f with how lanes share a channel of `order` states.
template <class F>
auto with_lanes(int order, F f) {
    if (order <= 4) return f(Lanes<1, 4, 4>{});
    if (order <= 8) return f(Lanes<2, 4, 4>{});
    if (order <= 16) return f(Lanes<4, 4, 4>{});
    if (order <= 32) return f(Lanes<4, 8, 4>{});
    return f(Lanes<4, 16, 4>{});
}

template <class L>
int slabs_of(const StateShape& s) {
    const int each = s.channels / s.groups;
    return (each + L::kSlab - 1) / L::kSlab;
}

// Waves of a pass without segments.
template <class L>
long long waves_of(const StateShape& s) {
    return static_cast<long long>(s.batch) * s.groups * slabs_of<L>(s) * L::W;
}

// The forward pass's.  With half of a wave for each SIMD (1024 of them), and not quite one, 8 lanes a
// channel are as many waves again, in place of segments: bfloat16 7 x 1000 x 2048, ragged (896 waves
// of 4 lanes) 56 us against 79 by 4 lanes, 4 x 4096 x 2048 (512) 229 against 241, 6 x 4096 x 2048
// (768) 354 against 365; 8 x 4096 x 2048 (1024) 427 against 366.  Orders 9 to 16 alone: it was not measured
// at others.
template <class F>
auto with_forward_lanes(const StateShape& s, F f) {
    if (s.order > 8 && s.order <= 16) {
        const long long waves = waves_of<Lanes<4, 4, 4>>(s);
        if (waves >= 512 && waves < 960) return f(Lanes<2, 8, 4>{});
    }
    return with_lanes(s.order, f);
}

// Slabs of the channels of a group, segments of the steps.
struct Cut {
    int slabs, segments, steps;  // steps of a segment, a multiple of kStateBlock
    int padded;                  // states of a channel in saved and workspace
    long long blocks;
};

// Workspace of the segments, for each sequence and segment: the end of the segment before it
// (segment 0: the given state) as padded rows of states a channel, and its own sums of dt; the
// backward pass has the gradient that leaves the segment instead.
struct Ends {
    float *states, *sums;
    __host__ __device__ Ends(float* workspace, const StateShape& s, const Cut& cut)
        : states(workspace),
          sums(workspace + static_cast<long long>(s.batch) * cut.segments * s.channels * cut.padded) {}
    static __device__ __forceinline__ long long row(const StateShape& s, const Cut& cut, int b, int segment,
                                                    int channel) {
        return (static_cast<long long>(b) * cut.segments + segment) * s.channels + channel;
    }
};

// Behind those: db and dc of a slab's channels, [slab][b][t][group][b's, c's] in padded rows; da,
// [b and segment][channel] in padded rows; dskip and ddelta_bias, two values for each b, segment
// and channel.
struct Parts {
    long long shared, da, pairs, count;  // offsets in floats; parts of da

    __host__ __device__ Parts(const StateShape& s, const Cut& cut) {
        count = static_cast<long long>(s.batch) * cut.segments;
        shared = cut.segments > 1 ? (count * s.channels * (cut.padded + 1) + 3) / 4 * 4 : 0;
        da = shared + static_cast<long long>(cut.slabs) * s.batch * s.n * s.groups * 2 * cut.padded;
        pairs = da + count * s.channels * cut.padded;
    }
    long long bytes(const StateShape& s) const { return 4 * (pairs + count * s.channels * 2); }
};

template <class T>
hipError_t launch_state_forward(const StateShape& s, const StateForward& a, const Cut& cut, hipStream_t stream);
template <class T>
hipError_t launch_state_backward(const StateShape& s, const StateBackward& a, const Cut& cut, hipStream_t stream);

}  // namespace thff
