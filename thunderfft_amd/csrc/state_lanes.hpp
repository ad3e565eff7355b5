// state_lanes.hpp -- how the lanes of a wave share the state space scan: LPC neighbouring lanes
// have a channel, S states each, and the wave 64 / LPC channels.  A lane also has one of every LPC
// steps of its channel, whose values it loads and whose sums over the states it ends up with.
#pragma once

#include "sequence_io.hpp"

namespace thff {

constexpr float kLog2e = 1.44269504f;

template <int Control>
__device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), Control, 0xf, 0xf, true));
}

// Values of the LPC lanes of a channel, to be had on all of them: of<K>() is the K-th lane's.  Among
// 4 lanes that is a modifier of the instruction that uses it; of 8, each half has a copy of the other.
template <int LPC>
struct Spread {
    static_assert(LPC == 4 || LPC == 8 || LPC == 16, "4, 8 or 16 lanes a channel");
    float low, high;

    __device__ __forceinline__ explicit Spread(float v) : low(v), high(v) {
        if constexpr (LPC == 8) {
            // 4 lanes back into the upper half of every 8, 4 on into the lower one.
            const int bits = __float_as_int(v);
            low = __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0x114, 0xf, 0xa, false));
            high = __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0x104, 0xf, 0x5, false));
        }
    }
    template <int K>
    __device__ __forceinline__ float of() const {
        if constexpr (LPC == 16) return moved<0x150 + K>(low);
        else return moved<K % 4 * 0x55>(K < 4 ? low : high);
    }
};

// The value of the lane mirrored within N lanes.
template <int N>
__device__ __forceinline__ float mirrored(float v) {
    return moved<N == 16 ? 0x140 : N == 8 ? 0x141 : N == 4 ? 0x1b : 0xb1>(v);
}

// Sums of v[k] over each LPC lanes: that of v[k] on the k-th lane.
template <int LPC>
__device__ __forceinline__ float sum_to_lanes(float (&v)[LPC], int lane) {
    if constexpr (LPC >= 16) {
        const bool high = lane & 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (high ? v[k + 8] : v[k]) + mirrored<16>(high ? v[k] : v[k + 8]);
    }
    if constexpr (LPC >= 8) {
        const bool high = lane & 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (high ? v[k + 4] : v[k]) + mirrored<8>(high ? v[k] : v[k + 4]);
    }
    const bool two = lane & 2, one = lane & 1;
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = (two ? v[k + 2] : v[k]) + mirrored<4>(two ? v[k] : v[k + 2]);
    return (one ? v[1] : v[0]) + mirrored<2>(one ? v[0] : v[1]);
}

// Sums of one and two over the lanes whose bit `Bit` differs: one's where the bit is 0, two's where
// it is 1.
template <int Bit>
__device__ __forceinline__ float sum_apart(float one, float two, int lane) {
    if constexpr (Bit == 5) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(one), __float_as_uint(two), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else if constexpr (Bit == 4) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(one), __float_as_uint(two), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
        static_assert(Bit == 3, "bits 5, 4 and 3");
        const bool high = lane & 8;
        return (high ? two : one) + moved<0x128>(high ? one : two);
    }
}

// Sums of v[0 ... N) over the channels of a wave, whose lanes have bits 5 down to log2(LPC): with each
// bit the values halve, until one is left or the bits are used up.  v[0 ...) are then those from
// ChannelSums::first(lane) on; lanes that differ in bits left have parts of the same ones.
template <int LPC, int N, int Bit = 5>
__device__ __forceinline__ void channel_sums(float* v, int lane) {
    if constexpr ((1 << Bit) >= LPC && N > 1) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = sum_apart<Bit>(v[i], v[i + N / 2], lane);
        channel_sums<LPC, N / 2, Bit - 1>(v, lane);
    }
}

// What is left of N values a lane, where the first of them belongs, how many lanes have parts of the
// same ones, and which of them the lane is.
template <int LPC, int N>
struct ChannelSums {
    static constexpr int kBits = LPC == 4 ? 4 : LPC == 8 ? 3 : 2;
    static constexpr int log2(int n) { return n == 1 ? 0 : 1 + log2(n / 2); }
    static constexpr int kApart = log2(N) < kBits ? log2(N) : kBits;  // bits that tell values apart
    static constexpr int kLeft = N >> kApart, kParts = 1 << (kBits - kApart);

    static __device__ __forceinline__ int first(int lane) {
        int at = 0;
#pragma unroll
        for (int k = 0; k < kApart; ++k) at += (lane >> (5 - k) & 1) * (N >> (k + 1));
        return at;
    }
    static __device__ __forceinline__ int part(int lane) { return lane / LPC % kParts; }
};

// log(1 + exp(v)) by e = exp(-|v|) and log(1 + e): u = 1 + e is rounded, and what is lost, e - (u - 1),
// changes the logarithm by its u-th part, of which 1 - e / 2 is near enough: 2^-26 of e at most.  The
// hardware's log is off by 2 units of its last place next to 1 too.  (A series for atanh takes 5
// instructions more.)
__device__ __forceinline__ float softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(v)), u = 1.0f + e;
    const float lost = (e - (u - 1.0f)) * fmaf(-0.5f, e, 1.0f);
    return __builtin_elementwise_maximum(v, 0.0f) + fmaf(__builtin_amdgcn_logf(u), 0.69314718f, lost);
}

__device__ __forceinline__ float opened(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * v));
}

// a log2(e), whose product with a dt is the power of two that a state keeps.  The lowest and highest values
// and infinities are taken as fp32's largest of their sign, so that a dt of 0 (a step behind the end, say)
// keeps the state, and what is 0 of a state that leaves nothing stays 0 times that; a NaN stays one.
__device__ __forceinline__ float rate_of(float a) {
    constexpr float kMost = 3.40282347e38f;
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(a * kLog2e, -kMost), kMost);
}

template <int N, class F, int K = 0>
__device__ __forceinline__ void each_step(F f) {
    if constexpr (K < N) {
        f(std::integral_constant<int, K>{});
        each_step<N, F, K + 1>(f);
    }
}

}  // namespace thff
