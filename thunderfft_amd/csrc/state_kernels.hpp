// state_kernels.hpp -- the kernels of the state space scan, one type of values a translation unit.
//
// A workgroup takes a slab of the channels of a group and walks over the steps of a segment of a
// sequence, one after the other: each lane holds S states of a channel in registers (state_lanes.hpp),
// and b and c, which all channels of the slab share, go through LDS in fp32.
//
// Where there are too few channels to fill the card, the steps are split into segments.  A first
// kernel takes each segment from a state of zero; as the decay of a segment is exp(a sum of dt),
// the states that the segments start from follow from those ends, in order.
//
// Instructions bound it: a state of a step takes 5 at least forward (dt a, its power, dt x b, and the
// sums of h and y) and 15 backward (those again and the gradients'), and takes 7.6 and 23.7 with what
// is once a step and channel, the addresses, LDS and the sums over channels.  bfloat16 8 x 4096 x 2048
// of 16 states (134 MB a tensor): forward 348 us, at a wave a SIMD, the VALU issuing in 67% of the
// cycles; backward 187 + 883 + 32 us by 4 segments, 84%.  1 x 65536 x 1024, forward: 202 + 288 us by
// 64 segments, 92% and 90%; all steps by one wave a channel 5.3 ms.  More waves a SIMD would need a
// backward tile in fewer than 256 registers.
#pragma once

#include <algorithm>
#include <type_traits>

#include "state_cut.hpp"
#include "state_lanes.hpp"

namespace thff {
namespace {

constexpr int kLanes = 256, kBlock = kStateBlock, kTile = kStateTile;

__device__ __forceinline__ int length_of(const int* lengths, int b, int n) {
    return lengths ? min(max(lengths[b], 0), n) : n;
}

template <class L>
struct Place {
    int lane, wave, sub;  // sub: of the channel's lanes
    int b, group, slab, segment;
    int base;  // the wave's first channel, or the group's last where the wave has none
    int in;    // the lane's from there, the group's last one again where it has none
    bool valid;

    __device__ __forceinline__ Place(const StateShape& s, const Cut& cut, long long block)
        : lane(threadIdx.x % 64), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)), sub(lane % L::LPC) {
        slab = static_cast<int>(block % cut.slabs);
        block /= cut.slabs;
        group = static_cast<int>(block % s.groups);
        block /= s.groups;
        segment = static_cast<int>(block % cut.segments);
        b = static_cast<int>(block / cut.segments);
        const int each = s.channels / s.groups, c = slab * L::kSlab + wave * L::kWave;
        valid = c + lane / L::LPC < each;
        base = group * each + min(c, each - 1);
        in = min(lane / L::LPC, max(each - 1 - c, 0));
    }
    __device__ __forceinline__ int channel() const { return base + in; }
};

// What lies at `at`, the same for all lanes of a wave, plus an offset of the lane's in elements.
template <class T>
__device__ __forceinline__ T& lane_at(T* at, unsigned offset) {
    return *reinterpret_cast<T*>(reinterpret_cast<char*>(const_cast<std::remove_const_t<T>*>(at)) +
                                 offset * static_cast<unsigned>(sizeof(T)));
}

__device__ __forceinline__ long long block_index() {
    return static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x;
}

// The lane's S states of rows of `order`, from `row` on; 0 where there is none.
template <class L>
__device__ __forceinline__ void load_states(float (&h)[L::S], const float* row, int sub, int order) {
#pragma unroll
    for (int i = 0; i < L::S; ++i) h[i] = sub * L::S + i < order ? row[sub * L::S + i] : 0.0f;
}

template <class L>
__device__ __forceinline__ void store_states(float* row, const float (&h)[L::S], int sub, int order) {
#pragma unroll
    for (int i = 0; i < L::S; ++i)
        if (sub * L::S + i < order) row[sub * L::S + i] = h[i];
}

// Padded rows: whole vectors.
template <class L>
__device__ __forceinline__ void load_padded(float (&h)[L::S], const float* row, int sub) {
    using V = float __attribute__((ext_vector_type(L::S)));
    const V v = *reinterpret_cast<const V*>(row + sub * L::S);
#pragma unroll
    for (int i = 0; i < L::S; ++i) h[i] = v[i];
}

template <class L>
__device__ __forceinline__ void store_padded(float* row, const float (&h)[L::S], int sub) {
    using V = float __attribute__((ext_vector_type(L::S)));
    V v;
#pragma unroll
    for (int i = 0; i < L::S; ++i) v[i] = h[i];
    __builtin_nontemporal_store(v, reinterpret_cast<V*>(row + sub * L::S));
}

// N values of a lane, LPC steps apart, from step t on, where `at` is: past the last step of n, the
// last one again.  offset: the lane's, of its step and channel.
template <int N, int LPC, class T>
__device__ __forceinline__ void load_steps(T (&v)[N], const T* at, unsigned offset, long long stride, int t, int sub, int n) {
    if (t + N * LPC <= n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = lane_at(at, offset);
            at += LPC * stride;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (&lane_at(at, offset))[(min(t + j * LPC + sub, n - 1) - sub - t) * stride];
    }
}

// Offsets of a lane's first step and channel in rows of each stride, and of its row and state of b's
// and c's; strides of more than kStateStride are refused.
template <class L>
struct Offsets {
    unsigned x, delta, gate, y, b, c;
    __device__ __forceinline__ Offsets(const StateShape& s, const Place<L>& p)
        : x(at(s.x_stride, p)), delta(at(s.delta_stride, p)), gate(at(s.gate_stride, p)), y(at(s.y_stride, p)),
          b(shared(s.b_stride, s, p)), c(shared(s.c_stride, s, p)) {}
    static __device__ __forceinline__ unsigned at(long long stride, const Place<L>& p) {
        return p.sub * static_cast<unsigned>(stride) + p.in;
    }
    static __device__ __forceinline__ unsigned shared(long long stride, const StateShape& s, const Place<L>& p) {
        return threadIdx.x / L::P * static_cast<unsigned>(stride) + min(static_cast<int>(threadIdx.x % L::P), s.order - 1);
    }
};

// b and c of N steps: loaded ahead into registers, then to LDS as [step][lane of a channel][b's, c's].
template <class T, class L, int N>
struct Shared {
    static constexpr int kEach = (N * L::P + L::kLanes - 1) / L::kLanes;
    using Rows = float[L::LPC][2 * L::S];
    static constexpr int kRows = L::kLanes / L::P;  // steps loaded at a time
    T b[kEach], c[kEach];

    // Steps from t0 on, where bs and cs are; b_at, c_at: the offsets of the lane's row of them and its state.
    template <bool Whole = false>
    __device__ __forceinline__ void load(const StateShape& s, const T* bs, const T* cs, unsigned b_at, unsigned c_at, int t0) {
        if (Whole || t0 + kEach * kRows <= s.n) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                b[e] = lane_at(bs, b_at);
                c[e] = lane_at(cs, c_at);
                bs += kRows * s.b_stride;
                cs += kRows * s.c_stride;
            }
        } else {
            const int row = threadIdx.x / L::P;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const long long t = min(t0 + e * kRows + row, s.n - 1) - row - t0;
                b[e] = (&lane_at(bs, b_at))[t * s.b_stride];
                c[e] = (&lane_at(cs, c_at))[t * s.c_stride];
            }
        }
    }
    // Zeros from step `end` on and for states that are none.
    __device__ __forceinline__ void store(const StateShape& s, Rows* to, int t0, int end) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = e * L::kLanes + threadIdx.x, st = i % L::P, t = i / L::P;
            if (N * L::P % L::kLanes != 0 && t >= N) break;
            const bool on = t0 + t < end && st < s.order;
            to[t][st / L::S][st % L::S] = on ? to_float<T>(b[e]) : 0.0f;
            to[t][st / L::S][L::S + st % L::S] = on ? to_float<T>(c[e]) : 0.0f;
        }
    }
};

template <int S>
__device__ __forceinline__ void load_shared(float (&b)[S], float (&c)[S], const float* row) {
    using V = float __attribute__((ext_vector_type(2 * S)));
    const V v = *reinterpret_cast<const V*>(row);
#pragma unroll
    for (int i = 0; i < S; ++i) {
        b[i] = v[i];
        c[i] = v[S + i];
    }
}

// Takes h through the segments from `from` on, `count` of them one after the other, `way` apart: each
// decays it by its sum of dt and adds its own end.  ends_of, sums_of: rows of the first one.  Where a is
// positive a segment's factor may be out of range though its product with h, or an h of zero, is not: its
// whole powers of two go to h's exponent (those past 300 take any h out of range, or to 0, by themselves).
template <class L>
__device__ __forceinline__ void fold(float (&h)[L::S], const float (&decay)[L::S], const float* ends_of, const float* sums_of,
                                     long long way, int count, int sub) {
    constexpr int kAtOnce = 8;  // loads under way together
    for (int k = 0; k < count; k += kAtOnce) {
        float own[kAtOnce][L::S], dt[kAtOnce];
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m) {
            const long long at = min(k + m, count - 1) * way;
            load_padded<L>(own[m], ends_of + at * L::P, sub);
            dt[m] = sums_of[at];
        }
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m) {
            if (k + m == count) break;
#pragma unroll
            for (int i = 0; i < L::S; ++i) {
                const float power = dt[m] * decay[i], whole = fminf(fmaxf(rintf(power), -300.0f), 300.0f);
                const float grown = __builtin_amdgcn_exp2f(power - whole) * h[i];
                h[i] = h[i] == 0.0f ? own[m][i] : __builtin_amdgcn_ldexpf(grown, static_cast<int>(whole)) + own[m][i];
            }
        }
    }
}

// The segment's end from a state of zero (the first segment: from the given one) where Only is
// `true`, for the segments but the last; its outputs otherwise.  Save: the states before every
// kTile-th step are kept.
//
// A block of steps that all count has no branches, so that the reads of LDS and the exponentials
// of one step are under way while those before it are worked on.  Lanes of no channel do as the
// last channel's, stores included.
template <class T, class L, bool Only, bool Save, bool Gate>
__global__ __launch_bounds__(L::kLanes) void state_forward(StateShape s, StateForward a, Cut cut) {
    constexpr int S = L::S, LPC = L::LPC, J = kBlock / LPC;
    __shared__ alignas(32) float bc[2][kBlock][LPC][2 * S];
    const long long block = block_index();
    if (block >= cut.blocks) return;
    const Place<L> p(s, cut, block);
    if (Only && p.segment + 1 == cut.segments) return;
    const int length = length_of(a.lengths, p.b, s.n), t0 = p.segment * cut.steps, t1 = min(t0 + cut.steps, s.n);
    const int end = min(length, t1);
    const long long first = p.b * static_cast<long long>(s.n) + t0;
    const Offsets<L> lane(s, p);
    const T* x = static_cast<const T*>(a.x) + first * s.x_stride + p.base;
    const T* delta = static_cast<const T*>(a.delta) + first * s.delta_stride + p.base;
    const T* gate = static_cast<const T*>(a.gate) + first * s.gate_stride + p.base;
    const T* bs = static_cast<const T*>(a.b) + first * s.b_stride + p.group * s.order;
    const T* cs = static_cast<const T*>(a.c) + first * s.c_stride + p.group * s.order;
    T* y = static_cast<T*>(a.y) + first * s.y_stride + p.base;
    const int channel = p.channel();
    float decay[S], h[S], sum = 0.0f;
    load_states<L>(decay, a.a + static_cast<long long>(channel) * s.order, p.sub, s.order);
#pragma unroll
    for (int i = 0; i < S; ++i) decay[i] = rate_of(decay[i]);
    const float skip = a.skip ? a.skip[channel] : 0.0f, bias = a.delta_bias ? a.delta_bias[channel] : 0.0f;

    int slot = p.b;
    if (a.slots) {
        slot = a.slots[p.b];
        if (slot < 0 || slot >= s.states) slot = -1;
    }
    const Ends ends(a.workspace, s, cut);
#pragma unroll
    for (int i = 0; i < S; ++i) h[i] = 0.0f;
    if (Only || cut.segments == 1) {
        if (p.segment == 0 && a.state_in && slot >= 0)
            load_states<L>(h, a.state_in + (static_cast<long long>(slot) * s.channels + channel) * s.order, p.sub, s.order);
        if (Only && p.segment == 0)
            store_padded<L>(ends.states + ends.row(s, cut, p.b, 0, channel) * L::P, h, p.sub);
    } else {
        load_padded<L>(h, ends.states + ends.row(s, cut, p.b, min(p.segment, 1), channel) * L::P, p.sub);
        fold<L>(h, decay, ends.states + ends.row(s, cut, p.b, 2, channel) * L::P, ends.sums + ends.row(s, cut, p.b, 1, channel),
                s.channels, p.segment - 1, p.sub);
    }
    const long long tiles = (s.n + kTile - 1) / kTile;
    float* saved = Save ? a.saved + (p.b * tiles * s.channels + channel) * L::P : nullptr;

    // Blocks of steps, LPC of them at a time, each lane with one.  Everything is under way early: what
    // the LPC steps have loaded is replaced by the next block's once it is used, dt and the gate of
    // the next LPC steps are worked out next to these steps' states, their b and c read from LDS, and
    // the next block's b and c go to LDS before this one ends.
    Shared<T, L, kBlock> ahead;
    T nx[J], nd[J], nz[J];
    struct Own {
        float x, dt, z;
    };
    const auto own_of = [&](int j, bool on) {
        Own o;
        o.x = on ? to_float<T>(nx[j]) : 0.0f;
        o.dt = softplus(to_float<T>(nd[j]) + bias);
        o.dt = on ? o.dt : 0.0f;
        o.z = 1.0f;
        if constexpr (Gate) {
            o.z = to_float<T>(nz[j]);
            o.z *= opened(o.z);
        }
        return o;
    };
    Own next = {};
    float b[2][LPC][S], c[2][LPC][S];
    int which = 0;
    const auto read = [&](int buffer, int j) {
#pragma unroll
        for (int k = 0; k < LPC; ++k) load_shared<S>(b[j & 1][k], c[j & 1][k], bc[buffer][j * LPC + k][p.sub]);
    };
    if (t0 < end) {
        ahead.load(s, bs, cs, lane.b, lane.c, t0);
        load_steps<J, LPC>(nx, x, lane.x, s.x_stride, t0, p.sub, s.n);
        load_steps<J, LPC>(nd, delta, lane.delta, s.delta_stride, t0, p.sub, s.n);
        if (Gate) load_steps<J, LPC>(nz, gate, lane.gate, s.gate_stride, t0, p.sub, s.n);
        ahead.store(s, bc[0], t0, end);
        next = own_of(0, t0 + p.sub < end);
    }
    // Whole: the block's steps and the next one's all count, and the loads' rows are all there.  Else the
    // LPC steps that begin behind the end are left out, of which there are many where n is small: 1024
    // sequences of one token (float, 2768 channels of 16 states) 366 us, 707 with all of them.
    const auto steps = [&](auto whole, int t) {
        constexpr bool kWhole = decltype(whole)::value;
        static_assert(J % 2 == 0, "the buffers of b and c go on from block to block");
        __syncthreads();
        read(which, 0);
        each_step<J>([&](auto j) {
            if (!kWhole && t + j * LPC >= end) return;
            if constexpr (j + 1 < J) read(which, j + 1);
            // The scheduler is kept to this order: left free it gathers the loads and the reads of LDS.
            __builtin_amdgcn_sched_barrier(0);
            const int now = t + j * LPC + p.sub;
            const Own own = next;
            sum += own.dt;
            if constexpr (j == 0) {
                bs += kBlock * s.b_stride;
                cs += kBlock * s.c_stride;
                if (kWhole) ahead.template load<true>(s, bs, cs, lane.b, lane.c, t + kBlock);
                else ahead.load(s, bs, cs, lane.b, lane.c, t + kBlock);
            }
            // The step a block on; past the last step, the last one again.
            const int skipped = kWhole ? kBlock : min(now + kBlock, s.n - 1) - now;
            nx[j] = lane_at(x + skipped * s.x_stride, lane.x);
            nd[j] = lane_at(delta + skipped * s.delta_stride, lane.delta);
            if (Gate) nz[j] = lane_at(gate + skipped * s.gate_stride, lane.gate);
            x += LPC * s.x_stride;
            delta += LPC * s.delta_stride;
            if (Gate) gate += LPC * s.gate_stride;
            next = own_of((j + 1) % J, kWhole || now + LPC < end);
            if constexpr (j == J - 1) ahead.store(s, bc[which ^ 1], t + kBlock, end);
            if constexpr (Save && j * LPC % kTile == 0) {
                if (kWhole || t + j * LPC < end)
                    store_padded<L>(saved + static_cast<long long>((t + j * LPC) / kTile) * s.channels * L::P, h, p.sub);
            }
            const Spread<LPC> dts(own.dt), us(own.dt * own.x);
            float part[LPC];
            each_step<LPC>([&](auto k) {
                const float d = dts.template of<k>(), v = us.template of<k>();
                part[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    h[i] = fmaf(__builtin_amdgcn_exp2f(d * decay[i]), h[i], v * b[j & 1][k][i]);
                    if (!Only) part[k] = fmaf(c[j & 1][k][i], h[i], part[k]);
                }
            });
            if constexpr (!Only) {
                const float v = fmaf(skip, own.x, sum_to_lanes<LPC>(part, p.lane)) * own.z;
                if (kWhole) lane_at(y, lane.y) = from_float<T>(v);
                else if (now < t1) lane_at(y, lane.y) = from_float<T>(now < end ? v : 0.0f);
                y += LPC * s.y_stride;
            }
        });
        which ^= 1;
    };
    int t = t0;
    constexpr int kAhead = std::max(kBlock, Shared<T, L, kBlock>::kEach * Shared<T, L, kBlock>::kRows);  // rows that a load may touch
    for (; t + 2 * kBlock <= end && t + kBlock + kAhead <= s.n; t += kBlock) steps(std::true_type{}, t);
    for (; t < end; t += kBlock) steps(std::false_type{}, t);
    t = min(t, t0 + (max(end - t0, 0) + LPC - 1) / LPC * LPC);  // what is left of the last block
    if constexpr (Only) {
        store_padded<L>(ends.states + ends.row(s, cut, p.b, p.segment + 1, channel) * L::P, h, p.sub);
        // The sum of the lanes' steps.
        float all[LPC];
#pragma unroll
        for (int k = 0; k < LPC; ++k) all[k] = sum;
        ends.sums[ends.row(s, cut, p.b, p.segment, channel)] = sum_to_lanes<LPC>(all, p.lane);
    } else {
        for (; t < t1; t += LPC, y += LPC * s.y_stride)
            if (t + p.sub < t1) lane_at(y, lane.y) = from_float<T>(0.0f);
        // Lanes of no channel, in other waves perhaps, have read the last channel's state too, which may be
        // replaced in place: after the barrier none still waits for it.
        if (a.state_out) __syncthreads();
        if (a.state_out && slot >= 0 && p.segment + 1 == cut.segments)
            store_states<L>(a.state_out + (static_cast<long long>(slot) * s.channels + channel) * s.order, h, p.sub, s.order);
    }
}

// ---- Backward. ----

// The gradient that leaves a segment towards its start, from one of zero behind it (the last
// segment: from dstate_out), where Only is `true`, for the segments but the first; the gradients
// otherwise.  Tiles go from the last to the first: the states of a tile are worked out again from the
// saved one and kept in registers with their decays, then the gradients go back over it.
//
// A tile whose steps and channels all count has no branches; of another one the LPC steps that begin
// behind the end are left out.
template <class T, class L, bool Only>
__global__ __launch_bounds__(L::kLanes, 2) void state_backward(StateShape s, StateBackward a, Cut cut) {
    constexpr int S = L::S, LPC = L::LPC, P = L::P, J = kTile / LPC;
    using Sums = ChannelSums<LPC, 2 * S>;
    __shared__ alignas(32) float bc[2][kTile][LPC][2 * S];
    __shared__ float sums[Only ? 1 : L::W * Sums::kParts][kTile][2 * P];
    const long long block = block_index();
    if (block >= cut.blocks) return;
    const Place<L> p(s, cut, block);
    if (Only && p.segment == 0) return;
    const int length = length_of(a.lengths, p.b, s.n), t0 = p.segment * cut.steps, t1 = min(t0 + cut.steps, s.n);
    const int end = min(length, t1);
    // The tile of the last step.
    const int from = end > t0 ? (end - 1 - t0) / kTile * kTile + t0 : t0 - kTile;
    const long long first = p.b * static_cast<long long>(s.n) + from, tiles = (s.n + kTile - 1) / kTile;
    const Offsets<L> lane(s, p);
    const T* x = static_cast<const T*>(a.x) + first * s.x_stride + p.base;
    const T* delta = static_cast<const T*>(a.delta) + first * s.delta_stride + p.base;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + first * s.gate_stride + p.base : nullptr;
    const T* dy = static_cast<const T*>(a.dy) + first * s.y_stride + p.base;
    const T* bs = static_cast<const T*>(a.b) + first * s.b_stride + p.group * s.order;
    const T* cs = static_cast<const T*>(a.c) + first * s.c_stride + p.group * s.order;
    T* dx = static_cast<T*>(a.dx) + first * s.x_stride + p.base;
    T* ddelta = static_cast<T*>(a.ddelta) + first * s.delta_stride + p.base;
    T* dgate = gate ? static_cast<T*>(a.dgate) + first * s.gate_stride + p.base : nullptr;
    const float* saved = a.saved + ((p.b * tiles + from / kTile) * s.channels + p.base) * P;
    const unsigned saved_at = p.in * P + p.sub * S;
    const int channel = p.channel();
    float decay[S], g[S], sum = 0.0f;
    load_states<L>(decay, a.a + static_cast<long long>(channel) * s.order, p.sub, s.order);
#pragma unroll
    for (int i = 0; i < S; ++i) decay[i] = rate_of(decay[i]);
    const float skip = a.skip ? a.skip[channel] : 0.0f, bias = a.delta_bias ? a.delta_bias[channel] : 0.0f;

    // g: the gradient of the state behind the steps that are done, from the steps behind it.
    const Ends ends(a.workspace, s, cut);
#pragma unroll
    for (int i = 0; i < S; ++i) g[i] = 0.0f;
    const int last = cut.segments - 1;
    if (p.segment == last) {
        if (a.dstate_out)
            load_states<L>(g, a.dstate_out + (static_cast<long long>(p.b) * s.channels + channel) * s.order, p.sub, s.order);
    } else if (!Only) {
        load_padded<L>(g, ends.states + ends.row(s, cut, p.b, last, channel) * P, p.sub);
        fold<L>(g, decay, ends.states + ends.row(s, cut, p.b, last - 1, channel) * P, ends.sums + ends.row(s, cut, p.b, last - 1, channel),
                -static_cast<long long>(s.channels), last - 1 - p.segment, p.sub);
    }
    // Lanes of no channel add nothing to the sums over channels.
#pragma unroll
    for (int i = 0; i < S; ++i) g[i] = p.valid ? g[i] : 0.0f;
    float da[S] = {}, dskip = 0.0f, dbias = 0.0f;
    const Parts parts(s, cut);
    float* shared_sums = a.workspace + parts.shared +
                         ((static_cast<long long>(p.slab) * s.batch + p.b) * s.n * s.groups + p.group) * 2 * P;
    const bool all_valid = (p.slab + 1) * static_cast<long long>(L::kSlab) <= s.channels / s.groups;

    // The values of the tile before are under way while a tile is worked on.
    Shared<T, L, kTile> ahead;
    T nx[J], nd[J], nz[J], ny[J];
    float nh[S];
    const auto load = [&](int t) {
        if (t < t0) return;
        ahead.load(s, bs, cs, lane.b, lane.c, t);
        if (!Only) load_padded<L>(nh, &lane_at(saved, saved_at), 0);
        load_steps<J, LPC>(nx, x, lane.x, s.x_stride, t, p.sub, s.n);
        load_steps<J, LPC>(nd, delta, lane.delta, s.delta_stride, t, p.sub, s.n);
        load_steps<J, LPC>(ny, dy, lane.y, s.y_stride, t, p.sub, s.n);
        if (gate) load_steps<J, LPC>(nz, gate, lane.gate, s.gate_stride, t, p.sub, s.n);
        bs -= kTile * s.b_stride;
        cs -= kTile * s.c_stride;
        saved -= static_cast<long long>(s.channels) * P;
        x -= kTile * s.x_stride;
        delta -= kTile * s.delta_stride;
        dy -= kTile * s.y_stride;
        if (gate) gate -= kTile * s.gate_stride;
    };
    // Stores a value of each of the lane's steps.
    const auto store = [&](auto whole, T* to, unsigned offset, long long stride, int t, const float (&v)[J]) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (decltype(whole)::value || (p.valid && t + j * LPC + p.sub < t1)) lane_at(to, offset) = from_float<T>(v[j]);
            to += LPC * stride;
        }
    };
    int which = 0;
    const auto steps = [&](auto whole, int t) {
        constexpr bool kWhole = decltype(whole)::value;
        ahead.store(s, bc[which], t, end);
        // Of the lane's step of each LPC.
        float xv[J], dt[J], along[J], raw[J], dyv[J], h[S];
        T zs[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool on = kWhole || (p.valid && t + j * LPC + p.sub < end);
            xv[j] = on ? to_float<T>(nx[j]) : 0.0f;
            raw[j] = to_float<T>(nd[j]) + bias;
            dt[j] = softplus(raw[j]);
            dt[j] = on ? dt[j] : 0.0f;
            dyv[j] = on ? to_float<T>(ny[j]) : 0.0f;
            along[j] = dyv[j];
            zs[j] = nz[j];
            sum += dt[j];
        }
        if (gate) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float z = to_float<T>(zs[j]);
                const bool on = kWhole || (p.valid && t + j * LPC + p.sub < end);
                along[j] = on ? dyv[j] * z * opened(z) : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < S; ++i) h[i] = nh[i];
        __syncthreads();
        load(t - kTile);
        float keep[kTile][S], before[Only ? 1 : kTile][S], inner[J];
        // Forward again from the saved state.
        each_step<J>([&](auto j) {
            inner[j] = 0.0f;
            if (!kWhole && t + j * LPC >= end) return;
            const Spread<LPC> dts(dt[j]), us(dt[j] * xv[j]);
            float out[LPC];
            each_step<LPC>([&](auto k) {
                constexpr int m = j * LPC + k;
                const float d = dts.template of<k>(), v = us.template of<k>();
                float b[S], c[S];
                load_shared<S>(b, c, bc[which][m][p.sub]);
                out[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    keep[m][i] = __builtin_amdgcn_exp2f(d * decay[i]);
                    if constexpr (!Only) {
                        before[m][i] = h[i];
                        h[i] = fmaf(keep[m][i], h[i], v * b[i]);
                        out[k] = fmaf(c[i], h[i], out[k]);
                    }
                }
            });
            if constexpr (!Only) inner[j] = fmaf(skip, xv[j], sum_to_lanes<LPC>(out, p.lane));
        });
        if constexpr (!Only) {
            if (gate) {
                float dz[J];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const float z = to_float<T>(zs[j]), f = opened(z);
                    const bool on = kWhole || t + j * LPC + p.sub < end;
                    dz[j] = on ? dyv[j] * inner[j] * fmaf(z * f, 1.0f - f, f) : 0.0f;
                }
                store(whole, dgate, lane.gate, s.gate_stride, t, dz);
            }
        }
        float ex[J], ed[J];
        // Left free, the scheduler begins with the way back early, for which there are no registers.
        __builtin_amdgcn_sched_barrier(0);
        each_step<J>([&](auto back) {
            constexpr int j = J - 1 - back;
            ex[j] = ed[j] = 0.0f;
            if (!kWhole && t + j * LPC >= end) return;
            const Spread<LPC> dts(dt[j]), us(dt[j] * xv[j]), alongs(along[j]);
            float du[LPC], de[LPC];
            each_step<LPC>([&](auto behind) {
                constexpr int k = LPC - 1 - behind, m = j * LPC + k;
                const float d = dts.template of<k>(), v = us.template of<k>(), dn = alongs.template of<k>();
                float b[S], c[S], both[2 * S];
                load_shared<S>(b, c, bc[which][m][p.sub]);
                du[k] = de[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const float lam = fmaf(dn, c[i], g[i]);
                    g[i] = keep[m][i] * lam;
                    if constexpr (!Only) {
                        both[i] = lam * v;
                        both[S + i] = dn * h[i];
                        du[k] = fmaf(lam, b[i], du[k]);
                        const float q = g[i] * before[m][i];
                        da[i] = fmaf(q, d, da[i]);
                        de[k] = fmaf(q, decay[i], de[k]);
                        h[i] = before[m][i];
                    }
                }
                if constexpr (!Only) {
                    channel_sums<LPC, 2 * S>(both, p.lane);
#pragma unroll
                    for (int l = 0; l < Sums::kLeft; ++l) {
                        const int at = Sums::first(p.lane) + l;
                        sums[p.wave * Sums::kParts + Sums::part(p.lane)][m][at / S * P + p.sub * S + at % S] = both[l];
                    }
                }
            });
            if constexpr (!Only) {
                const bool on = kWhole || t + j * LPC + p.sub < end;
                const float su = sum_to_lanes<LPC>(du, p.lane), se = sum_to_lanes<LPC>(de, p.lane) * (1.0f / kLog2e);
                // A dt of 0 keeps a state whatever the rate: the sum of q a may then be out of range, the slope is 0.
                const float slope = opened(raw[j]);
                ed[j] = fmaf(su, xv[j], slope == 0.0f ? 0.0f : se) * slope;
                ed[j] = on ? ed[j] : 0.0f;
                ex[j] = fmaf(su, dt[j], along[j] * skip);
                ex[j] = on ? ex[j] : 0.0f;
                dskip = fmaf(along[j], xv[j], dskip);
                dbias += ed[j];
            }
        });
        if constexpr (!Only) {
            store(whole, dx, lane.x, s.x_stride, t, ex);
            store(whole, ddelta, lane.delta, s.delta_stride, t, ed);
            dx -= kTile * s.x_stride;
            ddelta -= kTile * s.delta_stride;
            if (gate) dgate -= kTile * s.gate_stride;
            // The sums of all the waves' channels.
            __syncthreads();
            for (int e = threadIdx.x; e < kTile * 2 * P; e += L::kLanes) {
                const int m = e / (2 * P), at = e % (2 * P);
                float v = sums[0][m][at];
#pragma unroll
                for (int w = 1; w < L::W * Sums::kParts; ++w) v += sums[w][m][at];
                if (kWhole || t + m < end) shared_sums[static_cast<long long>(t + m) * s.groups * 2 * P + at] = v;
            }
        }
        which ^= 1;
    };
    load(from);
    int t = from;
    for (; t >= t0 && (t + kTile > end || !all_valid); t -= kTile) steps(std::false_type{}, t);
    for (; t >= t0; t -= kTile) steps(std::true_type{}, t);
    if (!p.valid) return;
    float all[LPC];
    const auto over_lanes = [&](float v) {
#pragma unroll
        for (int k = 0; k < LPC; ++k) all[k] = v;
        return sum_to_lanes<LPC>(all, p.lane);
    };
    const long long part = ends.row(s, cut, p.b, p.segment, channel);
    if constexpr (Only) {
        store_padded<L>(ends.states + part * P, g, p.sub);
        sum = over_lanes(sum);
        if (p.sub == 0) ends.sums[part] = sum;
    } else {
        // The pointers are a tile before the segment's first step.
        for (int t = max(from + kTile, t0); t + p.sub < t1; t += LPC) {
            const long long behind = t - t0 + kTile;
            lane_at(dx + behind * s.x_stride, lane.x) = from_float<T>(0.0f);
            lane_at(ddelta + behind * s.delta_stride, lane.delta) = from_float<T>(0.0f);
            if (gate) lane_at(dgate + behind * s.gate_stride, lane.gate) = from_float<T>(0.0f);
        }
        if (a.dstate_in && p.segment == 0)
            store_states<L>(a.dstate_in + (static_cast<long long>(p.b) * s.channels + channel) * s.order, g, p.sub, s.order);
        store_padded<L>(a.workspace + parts.da + part * P, da, p.sub);
        dskip = over_lanes(dskip);
        dbias = over_lanes(dbias);
        if (p.sub == 0) {
            a.workspace[parts.pairs + 2 * part] = dskip;
            a.workspace[parts.pairs + 2 * part + 1] = dbias;
        }
    }
}

// db and dc: the slabs' sums, in order; 0 behind a sequence's end.  Four states a lane.
template <class T>
__device__ __forceinline__ void add_shared(const StateShape& s, const StateBackward& a, const Cut& cut, const Parts& parts,
                                           long long block, long long blocks) {
    using V = float __attribute__((ext_vector_type(4)));
    const int row = 2 * cut.padded / 4;
    const long long count = static_cast<long long>(s.batch) * s.n * s.groups * row;
    const V* from = reinterpret_cast<const V*>(a.workspace + parts.shared);
    for (long long i = block * kLanes + threadIdx.x; i < count; i += blocks * kLanes) {
        const long long at = i / row, step = at / s.groups;
        const int group = static_cast<int>(at - step * s.groups), st = 4 * static_cast<int>(i - at * row);
        const int state = st % cut.padded, b = static_cast<int>(step / s.n);
        V sum = {};
        if (step - static_cast<long long>(b) * s.n < length_of(a.lengths, b, s.n)) {
            constexpr int kAtOnce = 8;  // loads under way together
            for (int k = 0; k < cut.slabs; k += kAtOnce) {
                V part[kAtOnce];
#pragma unroll
                for (int m = 0; m < kAtOnce; ++m) part[m] = from[min(k + m, cut.slabs - 1) * count + i];
#pragma unroll
                for (int m = 0; m < kAtOnce; ++m)
                    if (k + m < cut.slabs) sum += part[m];
            }
        }
        T* to = st < cut.padded ? static_cast<T*>(a.db) + step * s.b_stride : static_cast<T*>(a.dc) + step * s.c_stride;
#pragma unroll
        for (int m = 0; m < 4; ++m)
            if (state + m < s.order) to[group * s.order + state + m] = from_float<T>(sum[m]);
    }
}

// da, dskip and ddelta_bias: 32 sums a workgroup, 8 lanes a sum, each every 8th part.
__device__ __forceinline__ void add_weights(const StateShape& s, const StateBackward& a, const Cut& cut, const Parts& parts,
                                            long long block, long long blocks) {
    constexpr int kGroups = kLanes / 32;
    __shared__ float lds[kGroups][32];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const long long states = static_cast<long long>(s.channels) * cut.padded, sums = states + 2LL * s.channels;
    for (long long first = 32 * block; first < sums; first += 32 * blocks) {
        const long long i = first + lane;
        const bool pair = i >= states;
        const float* from = a.workspace + (pair ? parts.pairs + (i - states) : parts.da + i);
        const long long way = pair ? 2LL * s.channels : states;
        float sum = 0.0f;
        if (i < sums) {
#pragma unroll 8
            for (long long k = group; k < parts.count; k += kGroups) sum += from[k * way];
        }
        __syncthreads();
        lds[group][lane] = sum;
        __syncthreads();
        if (group != 0 || i >= sums) continue;
#pragma unroll
        for (int g = 1; g < kGroups; ++g) sum += lds[g][lane];
        if (!pair) {
            const long long c = i / cut.padded, state = i - c * cut.padded;
            if (state < s.order) a.da[c * s.order + state] = sum;
        } else {
            const long long c = (i - states) / 2;
            float* to = (i - states) % 2 ? a.ddelta_bias : a.dskip;
            if (to) to[c] = sum;
        }
    }
}

// What the backward pass's workgroups have left: the first `few` workgroups take the weights' sums.
template <class T>
__global__ __launch_bounds__(kLanes) void add_state_parts(StateShape s, StateBackward a, Cut cut, int few) {
    const Parts parts(s, cut);
    if (static_cast<int>(blockIdx.x) < few) add_weights(s, a, cut, parts, blockIdx.x, few);
    else add_shared<T>(s, a, cut, parts, blockIdx.x - few, gridDim.x - few);
}

// One step (n = 1: a token of each sequence): the states read and written once bound it, half 256 x
// 4096 of 16 states 22.2 us (126 MB, 5.7 TB/s), bfloat16 8 x 1024 3.5 us.  4 states a lane, Each lanes of them a channel, and Rows
// sequences one after the other, whose loads are all under way together and share a's.
template <class T, int Each, int Rows>
__global__ __launch_bounds__(kLanes, 6) void state_step(StateShape s, StateForward a) {
    const long long i = (block_index() * kLanes + threadIdx.x) / Each;
    const int b0 = static_cast<int>(i / s.channels), channel = static_cast<int>(i - static_cast<long long>(b0) * s.channels);
    if (b0 >= (s.batch + Rows - 1) / Rows) return;
    const int sub = threadIdx.x % Each, at = sub * 4, some = min(4, s.order - at);
    const int shared = channel / (s.channels / s.groups) * s.order + at;
    // Values of one lane's states, 0 where it has none.
    const auto load = [&](const auto* from) {
        using U = std::remove_const_t<std::remove_pointer_t<decltype(from)>>;
        pack<U, 4> v = {};
        if (some == 4) {
            v = load_pack<U, 4>(from);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < some) v[k] = from[k];
        }
        return v;
    };
    pack<float, 4> h[Rows];
    pack<T, 4> bv[Rows], cv[Rows];
    T x[Rows], delta[Rows], gate[Rows];
    long long state[Rows];
    int slot[Rows];
    bool on[Rows];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        // Sequences behind the last are the last, and not stored.
        const int b = min(b0 * Rows + r, s.batch - 1);
        slot[r] = a.slots ? a.slots[b] : b;
        if (a.slots && (slot[r] < 0 || slot[r] >= s.states)) slot[r] = -1;
        on[r] = length_of(a.lengths, b, 1) > 0;
        state[r] = (static_cast<long long>(slot[r]) * s.channels + channel) * s.order + at;
        x[r] = static_cast<const T*>(a.x)[b * s.x_stride + channel];
        delta[r] = static_cast<const T*>(a.delta)[b * s.delta_stride + channel];
        if (a.gate) gate[r] = static_cast<const T*>(a.gate)[b * s.gate_stride + channel];
        bv[r] = load(static_cast<const T*>(a.b) + b * s.b_stride + shared);
        cv[r] = load(static_cast<const T*>(a.c) + b * s.c_stride + shared);
    }
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        h[r] = pack<float, 4>{};
        if (a.state_in && slot[r] >= 0) h[r] = load(a.state_in + state[r]);
    }
    pack<float, 4> rate = load(a.a + static_cast<long long>(channel) * s.order + at);
#pragma unroll
    for (int k = 0; k < 4; ++k) rate[k] = rate_of(rate[k]);
    const float bias = a.delta_bias ? a.delta_bias[channel] : 0.0f, skip = a.skip ? a.skip[channel] : 0.0f;
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int b = b0 * Rows + r;
        const float xv = to_float<T>(x[r]), dt = softplus(to_float<T>(delta[r]) + bias), u = dt * xv;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float next = fmaf(__builtin_amdgcn_exp2f(dt * rate[k]), h[r][k], u * to_float<T>(bv[r][k]));
            if (on[r]) h[r][k] = next;
            if (k < some) sum = fmaf(to_float<T>(cv[r][k]), next, sum);
        }
        if constexpr (Each >= 2) sum += mirrored<2>(sum);
        if constexpr (Each >= 4) sum += mirrored<4>(sum);
        if constexpr (Each >= 8) sum += mirrored<8>(sum);
        if constexpr (Each >= 16) sum += mirrored<16>(sum);
        sum = fmaf(skip, xv, sum);
        if (a.gate) {
            const float z = to_float<T>(gate[r]);
            sum *= z * opened(z);
        }
        if (b >= s.batch) continue;
        if (sub == 0) static_cast<T*>(a.y)[b * s.y_stride + channel] = from_float<T>(on[r] ? sum : 0.0f);
        if (a.state_out && slot[r] >= 0) {
            // Few states through the caches, as the next token reads them soon; many past them.
            if (some == 4 && Rows > 1) {
                store_pack<float, 4>(a.state_out + state[r], h[r]);
            } else if (some == 4) {
                *reinterpret_cast<pack<float, 4>*>(a.state_out + state[r]) = h[r];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < some) a.state_out[state[r] + k] = h[r][k];
            }
        }
    }
}

}  // namespace
}  // namespace thff
