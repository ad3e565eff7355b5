// scan_last.hpp -- the gated recurrence on [batch][n][channels] values: one pass over the
// data.  A lane takes VEC neighbouring channels of S steps and composes them; the lanes and
// waves of a workgroup join theirs through LDS, and the workgroups through the chain.
//
// About 10 operations for 6 bytes forward (2-byte values): memory bounds it, and next to it the
// time from a tile's loads to its stores, in which its registers serve nobody else.  bfloat16
// 8 x 4096 x 2048: 85 us forward (403 MB, 4.8 TB/s) and 146 us backward (671 MB, 4.6 TB/s); the
// same tiles copied with no work between take 70 to 75 us forward.  Of the 10.4 us from a
// workgroup's start to the next one's in its place, 2.7 go to the draw and the first loads, 1.8
// until the last wave has its own, 1.7 to the chain, 1.4 to arithmetic and 2.8 pass between the
// two.  1 x 65536 x 1024 takes 108 us for the same bytes: 64 tiles of a column run side by side
// there, and each waits for the slowest of those before it.
#pragma once

#include <type_traits>

#include "scan_chain.hpp"

namespace thff {

// VEC channels and S steps a lane; CL lanes side by side along the channels, the other
// lanes of a wave and the W waves one behind the other along the steps.  C more waves draw
// tiles and wait for the chain, a lane for each channel or two: the others' registers hold
// nothing of it.  Occupancy: waves that a SIMD is to hold.
//
// 4 bytes a lane and row, 8 steps a lane forward and 4 backward are what 64 registers hold, so
// that two workgroups of 16 waves fill a compute unit: one loads while the other waits.  (16 steps
// at half the occupancy: 114 against 110 us at 1 x 65536 x 1024, 26 against 22.5 at
// 1 x 10000 x 1024.  Workgroups that go on to a next tile, its loads under way meanwhile: 101
// to 105 against 97 us at 8 x 4096 x 2048.)  The narrow tile's backward pass of 2-byte values does
// not quite fit, and has 40 bytes a lane in scratch memory.
template <int VEC_, int CL_, int S_, int W_, int C_, int Occupancy_>
struct Tile {
    static constexpr int VEC = VEC_, CL = CL_, S = S_, W = W_, C = C_;
    static constexpr int kOccupancy = Occupancy_, kLanes = 64 * (W + C);
    static constexpr int kChannels = VEC * CL;
    static constexpr int kSteps = W * (64 / CL) * S;
};
// Steps between the states that the forward pass saves for the backward pass.
constexpr int kSaved = 56;

// Joins the lanes' spans of a wave along the steps (lanes CL apart): `mine` becomes the span
// of everything up to and with this lane, the result is that of everything before it.
// Backward: later lanes come first.
template <int CL, bool Backward>
__device__ __forceinline__ Span join_lanes(Span& mine) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int d = CL; d < 64; d *= 2) {
        const int from = Backward ? lane + d : lane - d;
        const Span other = {__shfl(mine.a, from & 63), __shfl(mine.b, from & 63)};
        if (from >= 0 && from < 64) mine = then(other, mine);
    }
    Span before = {1.0f, 0.0f};
    if constexpr (CL < 64) {
        const int from = Backward ? lane + CL : lane - CL;
        const Span other = {__shfl(mine.a, from & 63), __shfl(mine.b, from & 63)};
        if (from >= 0 && from < 64) before = other;
    }
    return before;
}

// A lane's S rows of VEC values: `at`, the same for the wave (so that it stays in scalar
// registers), and the lane's own part of the offset.
template <int CL>
using LaneOffset = std::conditional_t<CL == 64, unsigned, long long>;

template <class L>
__device__ __forceinline__ LaneOffset<L::CL> lane_offset(long long stride) {
    const int lane = threadIdx.x % 64;
    if constexpr (L::CL == 64) return lane * L::VEC;
    return lane / L::CL * L::S * stride + lane % L::CL * L::VEC;
}

// A stride that the compiler sees anew each time: it would keep a multiple of it for every
// row, and has not so many registers.
__device__ __forceinline__ long long anew(long long stride) {
    asm volatile("" : "+s"(stride));
    return stride;
}

// A lane's rows: `inside` are steps of the sequence, the next ones up to `rows` lie in the
// tensor, and `some` of VEC channels.  full: all of the wave's are inside.
struct Inside {
    bool full;
    int inside, rows, some;
};

// Where not all is inside, a lane reads its last row instead of those past the tensor, and the
// last VEC channels instead of some of them and some that are not there, so that no load waits
// for another or for a branch; keep_inside() puts that right when all loads are under way.
template <class T, class L, class Offset>
__device__ __forceinline__ void load_steps(pack<T, L::VEC> (&to)[L::S], const T* at, Offset lane,
                                           long long stride, Inside in, int channels) {
    constexpr int VEC = L::VEC, S = L::S;
    stride = anew(stride);
    if (in.full) {
#pragma unroll
        for (int k = 0; k < S; ++k, at += stride) to[k] = load_pack<T, VEC>(at + lane);
        return;
    }
#pragma unroll
    for (int k = 0; k < S; ++k) to[k] = pack<T, VEC>{};
    if (in.inside <= 0 || in.some <= 0) return;  // nothing that is used
    const int shift = VEC - in.some;
    const T* p = at + lane;
    if (channels < VEC) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i >= shift) to[k][i] = p[i - shift];
            if (k < in.rows - 1) p += stride;
        }
    } else {
        p -= shift;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            to[k] = load_pack<T, VEC>(p);
            if (k < in.rows - 1) p += stride;
        }
    }
}

// Moves the channels of a vector that was read further back to its start, and puts `none` in the
// place of steps that are not inside.
template <class T, class L>
__device__ __forceinline__ void keep_inside(pack<T, L::VEC> (&v)[L::S], Inside in, T none) {
    static_assert(L::VEC <= 2, "a vector is cut after its first channel");
    if (in.full) return;
#pragma unroll
    for (int k = 0; k < L::S; ++k) {
        if (in.some < L::VEC) v[k][0] = v[k][L::VEC - 1];
        if (k >= in.inside) v[k] = none;
    }
}

// Stores row k of a lane's S; zeros past the sequence's end.
template <class T, int VEC>
__device__ __forceinline__ void store_step(T* at, pack<T, VEC> v, int k, Inside in) {
    if (in.full)
        store_pack<T, VEC>(at, v);
    else if (k < in.rows && in.some > 0)
        store_some<T, VEC>(at, k < in.inside ? v : pack<T, VEC>{}, in.some);
}

// Where a tile lies: the same on every lane.
template <class L, bool Backward>
struct Place {
    int tile, b, c0, len, column;

    // The workgroup's, the `drawn`-th of its column in the order of the chain.
    __device__ __forceinline__ Place(int drawn, const ScanShape& s, const int* lengths,
                                     const Chain& chain) {
        tile = Backward ? chain.tiles - 1 - drawn : drawn;
        column = chain.column();
        b = chain.by_slabs.quotient(column);
        c0 = (column - b * chain.slabs) * L::kChannels;
        len = length_of(lengths, b, s.n);
    }
    __device__ __forceinline__ int t0() const { return tile * L::kSteps; }
    // The lane's, whose first step is `sub` from the tile's.
    __device__ __forceinline__ Inside inside(const ScanShape& s, int wave, int sub) const {
        const int t = t0() + sub;
        return {t0() + (wave + 1) * (64 / L::CL) * L::S <= len && c0 + L::kChannels <= s.channels,
                max(0, min(L::S, len - t)), max(0, min(L::S, s.n - t)),
                max(0, min(L::VEC,
                           s.channels - c0 - static_cast<int>(threadIdx.x) % L::CL * L::VEC))};
    }
    // The first of the wave's rows.
    __device__ __forceinline__ long long row(const ScanShape& s, int wave) const {
        return static_cast<long long>(b) * s.n + t0() + wave * (64 / L::CL) * L::S;
    }
};

__device__ __forceinline__ long long saved_at(const ScanShape& s, int b, int t, int steps) {
    return (static_cast<long long>(b) * ((s.n + steps - 1) / steps) + t / steps) * s.channels;
}

// The waves that publish and wait for other tiles: spans of a tile's waves in
// `waves`, in the order of the chain, which become those of all waves before each, and the state
// that the tile starts from in `start`.
// state(p): where that of the chain's first tile is given for channel p.c0, or null.
template <class L, bool Backward, class State>
__device__ __forceinline__ void run_chain(const ScanShape& s, const int* lengths, const Chain& chain,
                                          Span (*waves)[L::kChannels], float* start,
                                          int ticket, State state) {
    constexpr int N = L::kChannels > 64 * L::C ? L::kChannels / (64 * L::C) : 1;
    const int lane = threadIdx.x - 64 * L::W, c = lane * N;
    const Place<L, Backward> p(ticket, s, lengths, chain);
    const bool mine = c < L::kChannels;
    // Every tile has its place in the chain, also past the sequence's end, where its span changes
    // nothing: that no wait depends on the lengths is worth more than the shorter chain.
    Link<N> link;
    link.words = chain.words + static_cast<long long>(p.column) * L::kChannels + c;
    link.step = static_cast<long long>(chain.columns) * L::kChannels;
    link.r = Backward ? chain.tiles - 1 - p.tile : p.tile;
    float given[N] = {};
    if (mine) {
        link.ask();
        const float* from = state(p);
#pragma unroll
        for (int v = 0; v < N; ++v)
            if (link.r == 0 && from && p.c0 + c + v < s.channels) given[v] = from[c + v];
    }
    __syncthreads();
    if (mine) {
        Span all[N];
#pragma unroll
        for (int v = 0; v < N; ++v) {
            // A wave's own span makes room for that of the waves before it; some at a time, for
            // want of registers.
            constexpr int kSome = L::W / 2;
            static_assert(L::W % 2 == 0, "two halves");
            all[v] = {1.0f, 0.0f};
#pragma unroll
            for (int w0 = 0; w0 < L::W; w0 += kSome) {
                Span each[kSome];
#pragma unroll
                for (int w = 0; w < kSome; ++w) each[w] = waves[w0 + w][c + v];
#pragma unroll
                for (int w = 0; w < kSome; ++w) {
                    waves[w0 + w][c + v] = all[v];
                    all[v] = then(all[v], each[w]);
                }
            }
        }
        float h[N];
        link.join(h, all, link.r + 1 < chain.tiles, given);
#pragma unroll
        for (int v = 0; v < N; ++v) start[c + v] = h[v];
    }
    __syncthreads();
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes, L::kOccupancy) void scan_last_forward(ScanShape s, ScanForward a,
                                                                  Chain chain) {
    constexpr int VEC = L::VEC, S = L::S, TL = 64 / L::CL;
    using Where = Place<L, false>;
    __shared__ Span waves[L::W][L::kChannels];
    __shared__ float start[L::kChannels];
    __shared__ int drawn;
    if (chain.block() >= chain.blocks) return;
    const bool chained = chain.tiles > 1;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int cl = lane % L::CL * VEC, sub = (wave * TL + lane / L::CL) * S;
    if (wave >= L::W) {
        const int ticket = chained ? draw_tile(chain, &drawn, L::W) : 0;
        run_chain<L, false>(s, a.lengths, chain, waves, start, ticket, [&](const Where& p) {
            const int row = state_row(s, a.slots, p.b);
            return a.state_in && row >= 0
                       ? a.state_in + static_cast<long long>(row) * s.channels + p.c0
                       : nullptr;
        });
        return;
    }
    const auto at_x = lane_offset<L>(s.x_stride), at_gate = lane_offset<L>(s.gate_stride),
               at_y = lane_offset<L>(s.y_stride);
    // The loads of the tile that it expects to draw go before the draw; they are done again if
    // it draws another.
    Where p(chained ? chain.expected() : 0, s, a.lengths, chain);
    pack<T, VEC> x[S], g[S];
    const auto load = [&] {
        const long long row = p.row(s, wave);
        const Inside in = p.inside(s, wave, sub);
        load_steps<T, L>(g, static_cast<const T*>(a.gate) + row * s.gate_stride + p.c0, at_gate,
                         s.gate_stride, in, s.channels);
        load_steps<T, L>(x, static_cast<const T*>(a.x) + row * s.x_stride + p.c0, at_x, s.x_stride,
                         in, s.channels);
    };
    load();
    if (chained) {
        const int ticket = draw_tile(chain, &drawn, L::W);
        if (ticket != chain.expected()) {
            p = Where(ticket, s, a.lengths, chain);
            load();
        }
    }
    const long long first = p.row(s, wave);
    const Inside in = p.inside(s, wave, sub);
    keep_inside<T, L>(g, in, open_gate<T>());
    keep_inside<T, L>(x, in, static_cast<T>(0.0f));
    float f[S][VEC], u[S][VEC];
    Span before[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) before[v] = {1.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < S; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Gate q = gate_of(to_float<T>(g[k][v]));
            f[k][v] = q.keep;
            u[k][v] = q.enter * to_float<T>(x[k][v]);
            before[v] = then_step(before[v], f[k][v], u[k][v]);
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Span mine = before[v];
        before[v] = join_lanes<L::CL, false>(mine);
        if (lane / L::CL == TL - 1) waves[wave][cl + v] = mine;
    }
    __syncthreads();
    __syncthreads();
    const int t = p.t0() + sub, row = state_row(s, a.slots, p.b);
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        h[v] = after(before[v], after(waves[wave][cl + v], start[cl + v]));
    T* y = static_cast<T*>(a.y) + first * s.y_stride + p.c0;
    const long long stride = anew(s.y_stride);
#pragma unroll
    for (int k = 0; k < S; ++k, y += stride) {
        if (k % 8 == 0 && a.saved && (t + k) % kSaved == 0 && t + k < s.n) {
            float* saved = a.saved + saved_at(s, p.b, t + k, kSaved) + p.c0 + cl;
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (v < in.some) saved[v] = h[v];
        }
        pack<T, VEC> out;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            h[v] = fmaf(f[k][v], h[v], u[k][v]);
            out[v] = from_float<T>(h[v]);
        }
        store_step<T, VEC>(y + at_y, out, k, in);
    }
    if (a.state_out && row >= 0 && (p.len > 0 ? t < p.len && p.len <= t + S : t == 0)) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < in.some)
                a.state_out[static_cast<long long>(row) * s.channels + p.c0 + cl + v] = h[v];
    }
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes, L::kOccupancy) void scan_last_backward(ScanShape s, ScanBackward a,
                                                                   Chain chain) {
    constexpr int VEC = L::VEC, S = L::S, W = L::W, TL = 64 / L::CL;
    static_assert(L::kSteps % kSaved == 0, "a tile starts from a saved state");
    using Where = Place<L, true>;
    // Spans of h, and of the gradient that goes back (the last wave's first).
    __shared__ Span waves[W][L::kChannels], back[W][L::kChannels];
    __shared__ float start[L::kChannels];
    __shared__ int drawn;
    if (chain.block() >= chain.blocks) return;
    const bool chained = chain.tiles > 1;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int cl = lane % L::CL * VEC, sub = (wave * TL + lane / L::CL) * S;
    if (wave >= W) {
        const int ticket = chained ? draw_tile(chain, &drawn, W) : 0;
        run_chain<L, true>(s, a.lengths, chain, back, start, ticket, [&](const Where& p) {
            return a.dstate_out
                       ? a.dstate_out + static_cast<long long>(p.b) * s.channels + p.c0
                       : nullptr;
        });
        return;
    }
    const auto at_x = lane_offset<L>(s.x_stride), at_gate = lane_offset<L>(s.gate_stride),
               at_y = lane_offset<L>(s.y_stride);
    Where p(chained ? chain.expected() : 0, s, a.lengths, chain);
    pack<T, VEC> x[S], g[S], dy[S];
    float h[VEC];  // the state before the tile
    const auto load = [&] {
        const long long row = p.row(s, wave);
        const Inside in = p.inside(s, wave, sub);
        load_steps<T, L>(g, static_cast<const T*>(a.gate) + row * s.gate_stride + p.c0, at_gate,
                         s.gate_stride, in, s.channels);
        load_steps<T, L>(x, static_cast<const T*>(a.x) + row * s.x_stride + p.c0, at_x, s.x_stride,
                         in, s.channels);
        load_steps<T, L>(dy, static_cast<const T*>(a.dy) + row * s.y_stride + p.c0, at_y, s.y_stride,
                         in, s.channels);
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            h[v] = p.t0() < p.len && v < in.some
                       ? a.saved[saved_at(s, p.b, p.t0(), kSaved) + p.c0 + cl + v]
                       : 0.0f;
    };
    load();
    if (chained) {
        const int ticket = draw_tile(chain, &drawn, W);
        if (ticket != chain.expected()) {
            p = Where(ticket, s, a.lengths, chain);
            load();
        }
    }
    const long long row = p.row(s, wave);
    const Inside in = p.inside(s, wave, sub);
    keep_inside<T, L>(g, in, open_gate<T>());
    keep_inside<T, L>(x, in, static_cast<T>(0.0f));
    keep_inside<T, L>(dy, in, static_cast<T>(0.0f));
    float f[S][VEC], enter[S][VEC], q[S][VEC];
    Span before[VEC], past[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) before[v] = past[v] = {1.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < S; ++k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Gate r = gate_of(to_float<T>(g[k][v]));
            f[k][v] = r.keep;
            enter[k][v] = r.enter;
            q[k][v] = to_float<T>(x[k][v]);
            before[v] = then_step(before[v], r.keep, r.enter * q[k][v]);
        }
    }
#pragma unroll
    for (int k = S - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            past[v] = then_step(past[v], f[k][v], f[k][v] * to_float<T>(dy[k][v]));
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Span mine = before[v], behind = past[v];
        before[v] = join_lanes<L::CL, false>(mine);
        past[v] = join_lanes<L::CL, true>(behind);
        if (lane / L::CL == TL - 1) waves[wave][cl + v] = mine;
        if (lane / L::CL == 0) back[W - 1 - wave][cl + v] = behind;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        for (int w = 0; w < wave; ++w) h[v] = after(waves[w][cl + v], h[v]);
        h[v] = after(before[v], h[v]);
    }
    // q becomes what lam is multiplied with for the gate's gradient.
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float in = q[k][v];
            q[k][v] = (h[v] - in) * (f[k][v] * enter[k][v]);
            h[v] = fmaf(f[k][v], h[v], enter[k][v] * in);
        }
    __syncthreads();
    const long long stride_x = anew(s.x_stride), stride_gate = anew(s.gate_stride);
    T* dx = static_cast<T*>(a.dx) + (row + S - 1) * s.x_stride + p.c0;
    T* dgate = static_cast<T*>(a.dgate) + (row + S - 1) * s.gate_stride + p.c0;
    float grad[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        grad[v] = after(past[v], after(back[W - 1 - wave][cl + v], start[cl + v]));
#pragma unroll
    for (int k = S - 1; k >= 0; --k, dx -= stride_x, dgate -= stride_gate) {
        pack<T, VEC> outx, outg;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float lam = to_float<T>(dy[k][v]) + grad[v];
            outx[v] = from_float<T>(enter[k][v] * lam);
            outg[v] = from_float<T>(q[k][v] * lam);
            grad[v] = f[k][v] * lam;
        }
        store_step<T, VEC>(dx + at_x, outx, k, in);
        store_step<T, VEC>(dgate + at_gate, outg, k, in);
    }
    if (a.dstate_in && p.tile == 0 && sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < in.some)
                a.dstate_in[static_cast<long long>(p.b) * s.channels + p.c0 + cl + v] = grad[v];
    }
}

}  // namespace thff
