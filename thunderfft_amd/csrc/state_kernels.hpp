// state_kernels.hpp -- the kernels of the state space scan, one type of values a translation unit.
//
// A workgroup takes a slab of the channels of a group and walks over the steps of a segment of a
// sequence, one after the other: each lane holds S states of a channel in registers (state_lanes.hpp),
// and b and c, which all channels of the slab share, go through LDS in fp32.
//
// Where there are too few channels to fill the card, the steps are split into segments.  A first
// kernel takes each segment from a state of zero; as the decay of a segment is exp(a sum of dt),
// the states that the segments start from follow from those ends, in order.
#pragma once

#include <algorithm>
#include <type_traits>

#include "state_cut.hpp"
#include "state_lanes.hpp"

namespace thff {
namespace {

constexpr int kWaves = kStateWaves, kLanes = 64 * kWaves, kBlock = kStateBlock, kTile = kStateTile;

__device__ __forceinline__ int length_of(const int* lengths, int b, int n) {
    return lengths ? min(max(lengths[b], 0), n) : n;
}

template <class L>
struct Place {
    int lane, wave, sub;  // sub: of the channel's lanes
    int b, group, slab, segment;
    int channel;  // the last one again where there is none
    bool valid;

    __device__ __forceinline__ Place(const StateShape& s, const Cut& cut, long long block)
        : lane(threadIdx.x % 64), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)), sub(lane % L::LPC) {
        slab = static_cast<int>(block % cut.slabs);
        block /= cut.slabs;
        group = static_cast<int>(block % s.groups);
        block /= s.groups;
        segment = static_cast<int>(block % cut.segments);
        b = static_cast<int>(block / cut.segments);
        const int each = s.channels / s.groups;
        const int c = slab * L::kSlab + wave * L::kWave + lane / L::LPC;
        valid = c < each;
        channel = group * each + min(c, each - 1);
    }
};

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

// b and c of N steps: loaded ahead into registers, then to LDS as [step][lane of a channel][b's, c's].
template <class T, class L, int N>
struct Shared {
    static constexpr int kEach = (N * L::P + kLanes - 1) / kLanes;
    using Rows = float[L::LPC][2 * L::S];
    T b[kEach], c[kEach];

    __device__ __forceinline__ void load(const StateShape& s, const T* bs, const T* cs, int t0) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = e * kLanes + threadIdx.x, st = min(i % L::P, s.order - 1);
            const long long t = min(t0 + i / L::P, s.n - 1);
            b[e] = bs[t * s.b_stride + st];
            c[e] = cs[t * s.c_stride + st];
        }
    }
    // Zeros from step `end` on and for states that are none.
    __device__ __forceinline__ void store(const StateShape& s, Rows* to, int t0, int end) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = e * kLanes + threadIdx.x, st = i % L::P, t = i / L::P;
            if (N * L::P % kLanes != 0 && t >= N) break;
            const bool on = t0 + t < end && st < s.order;
            to[t][st / L::S][st % L::S] = on ? to_float<T>(b[e]) : 0.0f;
            to[t][st / L::S][L::S + st % L::S] = on ? to_float<T>(c[e]) : 0.0f;
        }
    }
};

template <int S>
__device__ __forceinline__ void load_shared(float (&b)[S], float (&c)[S], const float* row) {
    using V = float __attribute__((ext_vector_type(S)));
    const V vb = *reinterpret_cast<const V*>(row), vc = *reinterpret_cast<const V*>(row + S);
#pragma unroll
    for (int i = 0; i < S; ++i) {
        b[i] = vb[i];
        c[i] = vc[i];
    }
}

// The segment's end from a state of zero (the first segment: from the given one) where Only is
// `true`, for the segments but the last; its outputs otherwise.
template <class T, class L, bool Only>
__global__ __launch_bounds__(kLanes) void state_forward(StateShape s, StateForward a, Cut cut) {
    constexpr int S = L::S, LPC = L::LPC, J = kBlock / LPC;
    __shared__ alignas(16) float bc[2][kBlock][LPC][2 * S];
    const long long block = block_index();
    if (block >= cut.blocks) return;
    const Place<L> p(s, cut, block);
    if (Only && p.segment + 1 == cut.segments) return;
    const int length = length_of(a.lengths, p.b, s.n), t0 = p.segment * cut.steps, t1 = min(t0 + cut.steps, s.n);
    const int end = min(length, t1);
    const long long first = p.b * static_cast<long long>(s.n);
    const int shared = p.group * s.order;
    const T* x = static_cast<const T*>(a.x) + first * s.x_stride + p.channel;
    const T* delta = static_cast<const T*>(a.delta) + first * s.delta_stride + p.channel;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + first * s.gate_stride + p.channel : nullptr;
    const T* bs = static_cast<const T*>(a.b) + first * s.b_stride + shared;
    const T* cs = static_cast<const T*>(a.c) + first * s.c_stride + shared;
    T* y = static_cast<T*>(a.y) + first * s.y_stride + p.channel;
    float decay[S], h[S], sum = 0.0f;
    load_states<L>(decay, a.a + static_cast<long long>(p.channel) * s.order, p.sub, s.order);
#pragma unroll
    for (int i = 0; i < S; ++i) decay[i] *= kLog2e;
    const float skip = a.skip ? a.skip[p.channel] : 0.0f, bias = a.delta_bias ? a.delta_bias[p.channel] : 0.0f;

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
            load_states<L>(h, a.state_in + (static_cast<long long>(slot) * s.channels + p.channel) * s.order, p.sub, s.order);
        if (Only && p.segment == 0 && p.valid)
            store_padded<L>(ends.states + ends.row(s, cut, p.b, 0, p.channel) * L::P, h, p.sub);
    } else {
        load_padded<L>(h, ends.states + ends.row(s, cut, p.b, min(p.segment, 1), p.channel) * L::P, p.sub);
        for (int k = 2; k <= p.segment; ++k) {
            float own[S];
            load_padded<L>(own, ends.states + ends.row(s, cut, p.b, k, p.channel) * L::P, p.sub);
            const float dt = ends.sums[ends.row(s, cut, p.b, k - 1, p.channel)];
#pragma unroll
            for (int i = 0; i < S; ++i) h[i] = fmaf(__builtin_amdgcn_exp2f(dt * decay[i]), h[i], own[i]);
        }
    }

    // The next block's values are under way while a block is worked on.
    Shared<T, L, kBlock> ahead;
    T nx[J], nd[J], nz[J];
    const auto load = [&](int t) {
        ahead.load(s, bs, cs, t);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const long long at = min(t + j * LPC + p.sub, s.n - 1);
            nx[j] = x[at * s.x_stride];
            nd[j] = delta[at * s.delta_stride];
            if (!Only && gate) nz[j] = gate[at * s.gate_stride];
        }
    };
    int which = 0;
    if (t0 < end) load(t0);
    int t = t0;
    for (; t < end; t += kBlock, which ^= 1) {
        ahead.store(s, bc[which], t, end);
        T xs[J], ds[J], zs[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            xs[j] = nx[j];
            ds[j] = nd[j];
            if (!Only && gate) zs[j] = nz[j];
        }
        __syncthreads();
        load(t + kBlock);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int now = t + j * LPC + p.sub;
            const bool on = now < end;
            const float xv = on ? to_float<T>(xs[j]) : 0.0f;
            const float dt = on ? softplus(to_float<T>(ds[j]) + bias) : 0.0f, u = dt * xv;
            if (!Only && j * LPC % kTile == 0 && a.saved && p.valid && t + j * LPC < end) {
                const long long tile = static_cast<long long>(p.b) * ((s.n + kTile - 1) / kTile) + (t + j * LPC) / kTile;
                store_padded<L>(a.saved + (tile * s.channels + p.channel) * L::P, h, p.sub);
            }
            sum += dt;
            float out[LPC];
            each_step<LPC>([&](auto k) {
                const float d = from_lane<LPC, k>(dt), v = from_lane<LPC, k>(u);
                float b[S], c[S];
                load_shared<S>(b, c, bc[which][j * LPC + k][p.sub]);
                out[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    h[i] = fmaf(__builtin_amdgcn_exp2f(d * decay[i]), h[i], v * b[i]);
                    if (!Only) out[k] = fmaf(c[i], h[i], out[k]);
                }
            });
            if constexpr (!Only) {
                float v = fmaf(skip, xv, sum_to_lanes<LPC>(out, p.lane));
                if (gate) {
                    const float z = to_float<T>(zs[j]);
                    v *= z * opened(z);
                }
                if (p.valid && now < t1) y[now * s.y_stride] = from_float<T>(on ? v : 0.0f);
            }
        }
    }
    if constexpr (Only) {
        if (!p.valid) return;
        store_padded<L>(ends.states + ends.row(s, cut, p.b, p.segment + 1, p.channel) * L::P, h, p.sub);
        // The sum of the lanes' steps.
        float all[LPC];
#pragma unroll
        for (int k = 0; k < LPC; ++k) all[k] = sum;
        sum = sum_to_lanes<LPC>(all, p.lane);
        if (p.sub == 0) ends.sums[ends.row(s, cut, p.b, p.segment, p.channel)] = sum;
    } else {
        if (!p.valid) return;
        for (; t < t1; t += LPC)
            if (t + p.sub < t1) y[(t + p.sub) * s.y_stride] = from_float<T>(0.0f);
        if (a.state_out && slot >= 0 && p.segment + 1 == cut.segments)
            store_states<L>(a.state_out + (static_cast<long long>(slot) * s.channels + p.channel) * s.order, h, p.sub, s.order);
    }
}

// ---- Backward. ----

// The gradient that leaves a segment towards its start, from one of zero behind it (the last
// segment: from dstate_out), where Only is `true`, for the segments but the first; the gradients
// otherwise.
template <class T, class L, bool Only>
__global__ __launch_bounds__(kLanes, 2) void state_backward(StateShape s, StateBackward a, Cut cut) {
    constexpr int S = L::S, LPC = L::LPC, P = L::P, J = kTile / LPC;
    using Sums = ChannelSums<LPC, 2 * S>;
    __shared__ alignas(16) float bc[2][kTile][LPC][2 * S];
    __shared__ float sums[Only ? 1 : kWaves][kTile][2 * P];
    const long long block = block_index();
    if (block >= cut.blocks) return;
    const Place<L> p(s, cut, block);
    if (Only && p.segment == 0) return;
    const int length = length_of(a.lengths, p.b, s.n), t0 = p.segment * cut.steps, t1 = min(t0 + cut.steps, s.n);
    const int end = min(length, t1);
    const long long first = p.b * static_cast<long long>(s.n);
    const int shared = p.group * s.order;
    const T* x = static_cast<const T*>(a.x) + first * s.x_stride + p.channel;
    const T* delta = static_cast<const T*>(a.delta) + first * s.delta_stride + p.channel;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + first * s.gate_stride + p.channel : nullptr;
    const T* dy = static_cast<const T*>(a.dy) + first * s.y_stride + p.channel;
    const T* bs = static_cast<const T*>(a.b) + first * s.b_stride + shared;
    const T* cs = static_cast<const T*>(a.c) + first * s.c_stride + shared;
    T* dx = static_cast<T*>(a.dx) + first * s.x_stride + p.channel;
    T* ddelta = static_cast<T*>(a.ddelta) + first * s.delta_stride + p.channel;
    T* dgate = gate ? static_cast<T*>(a.dgate) + first * s.gate_stride + p.channel : nullptr;
    const long long tiles = (s.n + kTile - 1) / kTile;
    const float* saved = a.saved + (p.b * tiles * s.channels + p.channel) * P;
    float decay[S], g[S], sum = 0.0f;
    load_states<L>(decay, a.a + static_cast<long long>(p.channel) * s.order, p.sub, s.order);
#pragma unroll
    for (int i = 0; i < S; ++i) decay[i] *= kLog2e;
    const float skip = a.skip ? a.skip[p.channel] : 0.0f, bias = a.delta_bias ? a.delta_bias[p.channel] : 0.0f;

    // g: the gradient of the state behind the steps that are done, from the steps behind it.
    const Ends ends(a.workspace, s, cut);
#pragma unroll
    for (int i = 0; i < S; ++i) g[i] = 0.0f;
    const int last = cut.segments - 1;
    if (p.segment == last) {
        if (a.dstate_out && p.valid)
            load_states<L>(g, a.dstate_out + (static_cast<long long>(p.b) * s.channels + p.channel) * s.order, p.sub, s.order);
    } else if (!Only) {
        load_padded<L>(g, ends.states + ends.row(s, cut, p.b, last, p.channel) * P, p.sub);
        for (int k = last - 1; k > p.segment; --k) {
            float own[S];
            load_padded<L>(own, ends.states + ends.row(s, cut, p.b, k, p.channel) * P, p.sub);
            const float dt = ends.sums[ends.row(s, cut, p.b, k, p.channel)];
#pragma unroll
            for (int i = 0; i < S; ++i) g[i] = fmaf(__builtin_amdgcn_exp2f(dt * decay[i]), g[i], own[i]);
        }
        if (!p.valid) {
#pragma unroll
            for (int i = 0; i < S; ++i) g[i] = 0.0f;
        }
    }
    float da[S] = {}, dskip = 0.0f, dbias = 0.0f;
    const Parts parts(s, cut);
    float* shared_sums = a.workspace + parts.shared +
                         ((static_cast<long long>(p.slab) * s.batch + p.b) * s.n * s.groups + p.group) * 2 * P;

    // The values of the tile before are under way while a tile is worked on.
    Shared<T, L, kTile> ahead;
    T nx[J], nd[J], nz[J], ny[J];
    float nh[S];
    const auto load = [&](int t) {
        t = max(t, 0);
        ahead.load(s, bs, cs, t);
        if (!Only) load_padded<L>(nh, saved + static_cast<long long>(t / kTile) * s.channels * P, p.sub);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const long long at = min(t + j * LPC + p.sub, s.n - 1);
            nx[j] = x[at * s.x_stride];
            nd[j] = delta[at * s.delta_stride];
            ny[j] = dy[at * s.y_stride];
            if (gate) nz[j] = gate[at * s.gate_stride];
        }
    };
    const int from = end > t0 ? (end - 1 - t0) / kTile * kTile + t0 : t0 - kTile;
    int which = 0;
    if (from >= t0) load(from);
    for (int t = from; t >= t0; t -= kTile, which ^= 1) {
        ahead.store(s, bc[which], t, end);
        // Of the lane's step of each LPC.
        float xv[J], dt[J], u[J], along[J], z[J], dyv[J], raw[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool on = p.valid && t + j * LPC + p.sub < end;
            xv[j] = on ? to_float<T>(nx[j]) : 0.0f;
            raw[j] = to_float<T>(nd[j]) + bias;
            dt[j] = on ? softplus(raw[j]) : 0.0f;
            u[j] = dt[j] * xv[j];
            dyv[j] = on ? to_float<T>(ny[j]) : 0.0f;
            along[j] = dyv[j];
            if (gate) {
                z[j] = to_float<T>(nz[j]);
                along[j] = on ? dyv[j] * z[j] * opened(z[j]) : 0.0f;
            }
            sum += dt[j];
        }
        float h[S];
#pragma unroll
        for (int i = 0; i < S; ++i) h[i] = Only ? 0.0f : nh[i];
        __syncthreads();
        load(t - kTile);
        float inner[J];
        float keep[kTile][S], before[Only ? 1 : kTile][S];
        // Forward again from the saved state.
        each_step<J>([&](auto j) {
            float out[LPC];
            each_step<LPC>([&](auto k) {
                constexpr int m = j * LPC + k;
                const float d = from_lane<LPC, k>(dt[j]), v = from_lane<LPC, k>(u[j]);
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
            if constexpr (!Only) {
                if (gate) inner[j] = fmaf(skip, xv[j], sum_to_lanes<LPC>(out, p.lane));
            }
        });
        each_step<J>([&](auto back) {
            constexpr int j = J - 1 - back;
            float du[LPC], de[LPC];
            each_step<LPC>([&](auto behind) {
                constexpr int k = LPC - 1 - behind, m = j * LPC + k;
                const float d = from_lane<LPC, k>(dt[j]), v = from_lane<LPC, k>(u[j]), dn = from_lane<LPC, k>(along[j]);
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
                    if (Sums::stores(p.lane)) {
#pragma unroll
                        for (int l = 0; l < Sums::kLeft; ++l) {
                            const int at = Sums::first(p.lane) + l;
                            sums[p.wave][m][at / S * P + p.sub * S + at % S] = both[l];
                        }
                    }
                }
            });
            if constexpr (!Only) {
                const int now = t + j * LPC + p.sub;
                const bool on = now < end;
                const float su = sum_to_lanes<LPC>(du, p.lane), se = sum_to_lanes<LPC>(de, p.lane) * (1.0f / kLog2e);
                const float dr = on ? fmaf(su, xv[j], se) * opened(raw[j]) : 0.0f;
                dskip = fmaf(along[j], xv[j], dskip);
                dbias += dr;
                if (p.valid && now < t1) {
                    dx[now * s.x_stride] = from_float<T>(on ? fmaf(su, dt[j], along[j] * skip) : 0.0f);
                    ddelta[now * s.delta_stride] = from_float<T>(dr);
                    if (gate) {
                        const float f = opened(z[j]);
                        dgate[now * s.gate_stride] =
                            from_float<T>(on ? dyv[j] * inner[j] * fmaf(z[j] * f, 1.0f - f, f) : 0.0f);
                    }
                }
            }
        });
        if constexpr (!Only) {
            // The sums of the waves' channels.
            __syncthreads();
            for (int e = threadIdx.x; e < kTile * 2 * P; e += kLanes) {
                const int m = e / (2 * P), at = e % (2 * P);
                float v = sums[0][m][at];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) v += sums[w][m][at];
                if (t + m < end) shared_sums[static_cast<long long>(t + m) * s.groups * 2 * P + at] = v;
            }
        }
    }
    if (!p.valid) return;
    float all[LPC];
    const auto over_lanes = [&](float v) {
#pragma unroll
        for (int k = 0; k < LPC; ++k) all[k] = v;
        return sum_to_lanes<LPC>(all, p.lane);
    };
    const long long row = ends.row(s, cut, p.b, p.segment, p.channel);
    if constexpr (Only) {
        store_padded<L>(ends.states + row * P, g, p.sub);
        sum = over_lanes(sum);
        if (p.sub == 0) ends.sums[row] = sum;
    } else {
        for (int t = max(from + kTile, t0) + p.sub; t < t1; t += LPC) {
            dx[t * s.x_stride] = from_float<T>(0.0f);
            ddelta[t * s.delta_stride] = from_float<T>(0.0f);
            if (gate) dgate[t * s.gate_stride] = from_float<T>(0.0f);
        }
        if (a.dstate_in && p.segment == 0)
            store_states<L>(a.dstate_in + (static_cast<long long>(p.b) * s.channels + p.channel) * s.order, g, p.sub, s.order);
        store_padded<L>(a.workspace + parts.da + row * P, da, p.sub);
        dskip = over_lanes(dskip);
        dbias = over_lanes(dbias);
        if (p.sub == 0) {
            a.workspace[parts.pairs + 2 * row] = dskip;
            a.workspace[parts.pairs + 2 * row + 1] = dbias;
        }
    }
}

// db and dc: the slabs' sums, in order; 0 behind a sequence's end.
template <class T>
__global__ __launch_bounds__(kLanes) void add_shared(StateShape s, StateBackward a, Cut cut) {
    const Parts parts(s, cut);
    const long long row = 2LL * cut.padded, count = static_cast<long long>(s.batch) * s.n * s.groups * row;
    for (long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x; i < count;
         i += static_cast<long long>(gridDim.x) * kLanes) {
        const long long at = i / row, step = at / s.groups;
        const int group = static_cast<int>(at - step * s.groups), st = static_cast<int>(i - at * row);
        const int state = st % cut.padded, b = static_cast<int>(step / s.n);
        if (state >= s.order) continue;
        float sum = 0.0f;
        if (step - static_cast<long long>(b) * s.n < length_of(a.lengths, b, s.n))
            for (int k = 0; k < cut.slabs; ++k) sum += a.workspace[parts.shared + k * count + i];
        const int column = group * s.order + state;
        if (st < cut.padded) static_cast<T*>(a.db)[step * s.b_stride + column] = from_float<T>(sum);
        else static_cast<T*>(a.dc)[step * s.c_stride + column] = from_float<T>(sum);
    }
}

// da, dskip and ddelta_bias: 32 sums a workgroup, 32 lanes a sum, each every 32nd part.
__global__ __launch_bounds__(1024) void add_weights(StateShape s, StateBackward a, Cut cut, long long count) {
    __shared__ float lds[32][33];
    const Parts parts(s, cut);
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const long long states = static_cast<long long>(s.channels) * cut.padded, sums = states + 2LL * s.channels;
    for (long long first = 32LL * blockIdx.x; first < sums; first += 32LL * gridDim.x) {
        const auto value = [&](long long i, long long part) {
            return i < states ? a.workspace[parts.da + part * states + i]
                              : a.workspace[parts.pairs + part * 2 * s.channels + (i - states)];
        };
        float sum = 0.0f;
        if (first + lane < sums)
            for (long long k = group; k < count; k += 32) sum += value(first + lane, k);
        __syncthreads();
        lds[group][lane] = sum;
        __syncthreads();
        sum = lds[lane][group];
#pragma unroll
        for (int m = 1; m < 32; m *= 2) sum += __shfl_xor(sum, m);
        const long long i = first + group;
        if (lane != 0 || i >= sums) continue;
        if (i < states) {
            const long long c = i / cut.padded, state = i - c * cut.padded;
            if (state < s.order) a.da[c * s.order + state] = sum;
        } else {
            const long long c = (i - states) / 2;
            float* to = (i - states) % 2 ? a.ddelta_bias : a.dskip;
            if (to) to[c] = sum;
        }
    }
}

// One step (n = 1: a token of each sequence): 4 states a lane, Lanes of them a channel.
template <class T, int Lanes>
__global__ __launch_bounds__(kLanes) void state_step(StateShape s, StateForward a) {
    const long long i = (block_index() * kLanes + threadIdx.x) / Lanes;
    const int b = static_cast<int>(i / s.channels), channel = static_cast<int>(i - static_cast<long long>(b) * s.channels);
    if (b >= s.batch) return;
    const int sub = threadIdx.x % Lanes, at = sub * 4, some = min(4, s.order - at);
    int slot = b;
    if (a.slots) {
        slot = a.slots[b];
        if (slot < 0 || slot >= s.states) slot = -1;
    }
    const bool on = length_of(a.lengths, b, 1) > 0;
    const long long state = (static_cast<long long>(slot) * s.channels + channel) * s.order + at;
    const int shared = channel / (s.channels / s.groups) * s.order + at;
    const float* decay = a.a + static_cast<long long>(channel) * s.order + at;
    const T* bs = static_cast<const T*>(a.b) + b * s.b_stride + shared;
    const T* cs = static_cast<const T*>(a.c) + b * s.c_stride + shared;
    pack<float, 4> h = {}, rate = {};
    pack<T, 4> bv = {}, cv = {};
    const bool stored = a.state_in && slot >= 0;
    if (some == 4) {
        if (stored) h = load_pack<float, 4>(a.state_in + state);
        rate = load_pack<float, 4>(decay);
        bv = load_pack<T, 4>(bs);
        cv = load_pack<T, 4>(cs);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < some) {
                if (stored) h[k] = a.state_in[state + k];
                rate[k] = decay[k];
                bv[k] = bs[k];
                cv[k] = cs[k];
            }
    }
    const float x = to_float<T>(static_cast<const T*>(a.x)[b * s.x_stride + channel]);
    const float raw = to_float<T>(static_cast<const T*>(a.delta)[b * s.delta_stride + channel]);
    const float z = a.gate ? to_float<T>(static_cast<const T*>(a.gate)[b * s.gate_stride + channel]) : 0.0f;
    const float dt = softplus(raw + (a.delta_bias ? a.delta_bias[channel] : 0.0f)), u = dt * x;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float next = fmaf(__builtin_amdgcn_exp2f(dt * (rate[k] * kLog2e)), h[k], u * to_float<T>(bv[k]));
        if (on) h[k] = next;
        if (k < some) sum = fmaf(to_float<T>(cv[k]), next, sum);
    }
    if constexpr (Lanes >= 2) sum += mirrored<2>(sum);
    if constexpr (Lanes >= 4) sum += mirrored<4>(sum);
    if constexpr (Lanes >= 8) sum += mirrored<8>(sum);
    if constexpr (Lanes >= 16) sum += mirrored<16>(sum);
    if (a.skip) sum = fmaf(a.skip[channel], x, sum);
    if (a.gate) sum *= z * opened(z);
    if (sub == 0) static_cast<T*>(a.y)[b * s.y_stride + channel] = from_float<T>(on ? sum : 0.0f);
    if (a.state_out && slot >= 0) {
        // Through the caches: the next token reads it soon.
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < some) a.state_out[state + k] = h[k];
    }
}

}  // namespace
}  // namespace thff
