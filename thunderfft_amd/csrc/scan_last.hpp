// scan_last.hpp -- the gated recurrence on [batch][n][channels] values: one pass over the
// data, the long axis split into tiles that many workgroups take at once.
//
// A step is h -> f h + u with u = (1 - f) x.  Steps compose: (A, B) then (f, u) is
// (f A, f B + u).  A lane takes VEC neighbouring channels of S steps and composes them; the
// lanes and waves of a workgroup join theirs through LDS, and a tile's (A, B) is published
// for the tiles behind it.  Every kGroup-th tile, the first one among them, publishes the
// state after it instead; a tile starts from the last such state before it, led through the
// (A, B) of the tiles in between, always in this order, so that the result does not depend
// on timing.  The backward pass goes the same way from the last step to the first, with
// c -> f (dy + c), c the gradient that reaches a step from the steps behind it.
//
// Published words are 64 bits, (A, B) or (0, state), and empty ones all ones: each is
// valid as soon as it is seen, without fences.  Workgroups draw tiles from a counter,
// first steps first, and publish before they wait, and wait only for tiles drawn earlier,
// which running workgroups hold: every wait ends.
#pragma once

#include <type_traits>

#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {

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

__device__ __forceinline__ int length_of(const int* lengths, int b, int n) {
    return lengths ? min(max(lengths[b], 0), n) : n;
}

// Row of the state pool for sequence b, or -1 (none).
__device__ __forceinline__ int state_row(const ScanShape& s, const int* slots, int b) {
    if (!slots) return b;
    const int row = slots[b];
    return row >= 0 && row < s.states ? row : -1;
}

// Steps between the states that the forward pass saves for the backward pass.
constexpr int kSavedSteps = 64;
constexpr int kGroup = 16;

// (A, B) of some steps: h -> A h + B.
struct Span {
    float a, b;
};

__device__ __forceinline__ Span then(Span first, Span second) {
    return {first.a * second.a, fmaf(second.a, first.b, second.b)};
}

__device__ __forceinline__ float after(Span s, float h) { return fmaf(s.a, h, s.b); }

using Word = unsigned long long;
constexpr Word kEmpty = ~0ull;

__device__ __forceinline__ void publish(Word* to, Span s) {
    // The one NaN that looks empty is replaced by another.
    unsigned a = __float_as_uint(s.a);
    if (a == ~0u) a = 0x7fc00000u;
    __hip_atomic_store(to, a | static_cast<Word>(__float_as_uint(s.b)) << 32, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ Word look(const Word* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ Span span_of(Word w) {
    return {__uint_as_float(static_cast<unsigned>(w)), __uint_as_float(static_cast<unsigned>(w >> 32))};
}

// The workspace: a counter, then a word for every channel of every tile.
struct Chain {
    unsigned* drawn;
    Word* words;
    int slabs, tiles;  // tiles along the channels, along the steps
    unsigned total;    // batch * slabs * tiles
};
constexpr long long kChainHead = 128;

// VEC channels and S steps a lane; CL lanes side by side along the channels, the other
// lanes of a wave and the W waves one behind the other along the steps.
template <int VEC_, int CL_, int S_, int W_>
struct Tile {
    static constexpr int VEC = VEC_, CL = CL_, S = S_, W = W_;
    static constexpr int kChannels = VEC * CL;
    static constexpr int kSubs = W * (64 / CL);
    static constexpr int kSteps = kSubs * S;
    static constexpr int kLanes = 64 * W;
};

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

// What the r-th tile of a column's chain starts from, put into `items` for the whole
// workgroup: for r = 0 the state given (`first`, `some` values, or null for zeros), else
// the last published state before the tile and the spans of the tiles in between, an item
// for each lane along the steps to wait for.  words: the chain's first tile; step: words
// from a tile to the next.
template <class L>
__device__ __forceinline__ void gather(const float* first, int some, const Word* words,
                                       long long step, int r, Span (*items)[L::kChannels]) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int sub = wave * (64 / L::CL) + lane / L::CL, c = lane % L::CL * L::VEC;
    if (r == 0) {
        // Through LDS, so that it has been read before anyone stores a last state there.
        if (sub == 0) {
#pragma unroll
            for (int v = 0; v < L::VEC; ++v)
                items[0][c + v] = {0.0f, first && v < some ? first[v] : 0.0f};
        }
        return;
    }
    const int base = (r - 1) / kGroup * kGroup;
    for (int item = sub; item < r - base; item += L::kSubs) {
        const Word* at = words + (base + item) * step + c;
        Word w[L::VEC];
        bool all;
        do {
            all = true;
#pragma unroll
            for (int v = 0; v < L::VEC; ++v) w[v] = look(at + v);
#pragma unroll
            for (int v = 0; v < L::VEC; ++v) all = all && static_cast<unsigned>(w[v]) != ~0u;
        } while (!all);
#pragma unroll
        for (int v = 0; v < L::VEC; ++v) items[item][c + v] = span_of(w[v]);
    }
}

// The state at the start of the r-th tile of the chain, for the channel at `c`.
template <class L>
__device__ __forceinline__ float start_of(int r, int c, const Span (*items)[L::kChannels]) {
    float h = items[0][c].b;
    const int count = r == 0 ? 1 : r - (r - 1) / kGroup * kGroup;
    for (int i = 1; i < count; ++i) h = after(items[i][c], h);
    return h;
}

template <class T>
__device__ __forceinline__ T open_gate() {
    return static_cast<T>(__builtin_inff());
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

// `inside` of the rows, and `some` values of each; `none` in the place of the others.
template <class T, class L, class Offset>
__device__ __forceinline__ void load_steps(pack<T, L::VEC> (&to)[L::S], const T* at, Offset lane,
                                           long long stride, bool full, int inside, int some,
                                           T none) {
    if (full) {
#pragma unroll
        for (int k = 0; k < L::S; ++k) to[k] = load_pack<T, L::VEC>(at + k * stride + lane);
    } else {
#pragma unroll
        for (int k = 0; k < L::S; ++k) {
            to[k] = none;
            if (k < inside && some > 0) to[k] = load_some<T, L::VEC>(at + k * stride + lane, some);
        }
    }
}

// Stores S rows, `rows` of them in the tensor, zeros from `inside` on.
template <class T, class L, class Offset>
__device__ __forceinline__ void store_steps(T* at, Offset lane, long long stride,
                                            const pack<T, L::VEC> (&from)[L::S], bool full,
                                            int inside, int rows, int some) {
    if (full) {
#pragma unroll
        for (int k = 0; k < L::S; ++k) store_pack<T, L::VEC>(at + k * stride + lane, from[k]);
    } else {
#pragma unroll
        for (int k = 0; k < L::S; ++k)
            if (k < rows && some > 0)
                store_some<T, L::VEC>(at + k * stride + lane,
                                      k < inside ? from[k] : pack<T, L::VEC>{}, some);
    }
}

// Draws a tile.
__device__ __forceinline__ unsigned draw(const Chain& chain) {
    return __hip_atomic_fetch_add(chain.drawn, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes, 4) void scan_last_forward(ScanShape s, ScanForward a,
                                                                  Chain chain) {
    constexpr int VEC = L::VEC, S = L::S, TL = 64 / L::CL;
    __shared__ Span waves[L::W][L::kChannels];
    __shared__ Span items[kGroup][L::kChannels];
    __shared__ unsigned drawn;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int sub = wave * TL + lane / L::CL, cl = lane % L::CL * VEC;
    const auto at_x = lane_offset<L>(s.x_stride), at_gate = lane_offset<L>(s.gate_stride),
               at_y = lane_offset<L>(s.y_stride);
    const bool chained = chain.tiles > 1;
    const int columns = s.batch * chain.slabs;

    unsigned ticket = blockIdx.x;
    if (chained) {
        if (threadIdx.x == 0) drawn = draw(chain);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(drawn);
        __syncthreads();
    }
    while (ticket < chain.total) {
        unsigned next = 0;
        if (chained && threadIdx.x == 0) next = draw(chain);
        const int tile = ticket / columns, column = ticket % columns;
        const int b = column / chain.slabs, c0 = column % chain.slabs * L::kChannels, c = c0 + cl;
        const int some = max(0, min(VEC, s.channels - c));
        const int len = length_of(a.lengths, b, s.n);
        const int t0 = tile * L::kSteps, t = t0 + sub * S;
        const int rows = max(0, min(S, s.n - t)), inside = max(0, min(S, len - t));
        const long long row = static_cast<long long>(b) * s.n + t0 + wave * TL * S;  // the wave's first
        T* y = static_cast<T*>(a.y) + row * s.y_stride + c0;
        const bool full = t0 + L::kSteps <= len && c0 + L::kChannels <= s.channels;
        // A tile that lies past the sequence's end has zeros to write and no part in the chain.
        const bool part = t0 < len || tile == 0;
        pack<T, VEC> x[S], g[S];
        float f[S][VEC], u[S][VEC];
        Span mine[VEC], before[VEC];
        if (part) {
            load_steps<T, L>(g, static_cast<const T*>(a.gate) + row * s.gate_stride + c0, at_gate, s.gate_stride,
                             full, inside, some, open_gate<T>());
            load_steps<T, L>(x, static_cast<const T*>(a.x) + row * s.x_stride + c0, at_x, s.x_stride,
                             full, inside, some, static_cast<T>(0.0f));
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                mine[v] = {1.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    const Gate q = gate_of(to_float<T>(g[k][v]));
                    f[k][v] = q.keep;
                    u[k][v] = q.enter * to_float<T>(x[k][v]);
                    mine[v] = then(mine[v], {f[k][v], u[k][v]});
                }
                before[v] = join_lanes<L::CL, false>(mine[v]);
                if (lane / L::CL == TL - 1) waves[wave][cl + v] = mine[v];
            }
        }
        if (chained && threadIdx.x == 0) drawn = next;
        __syncthreads();
        if (chained) next = __builtin_amdgcn_readfirstlane(drawn);
        Word* words = chain.words + static_cast<long long>(column) * L::kChannels;
        const long long step = static_cast<long long>(columns) * L::kChannels;
        const bool gives_state = tile % kGroup == 0;
        const bool later = chained && t0 + L::kSteps < len;  // a tile waits for this one
        const int srow = state_row(s, a.slots, b);
        const long long state = static_cast<long long>(srow) * s.channels + c;
        Span ahead[VEC];  // of the waves before this one
        if (part) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ahead[v] = {1.0f, 0.0f};
                for (int w = 0; w < wave; ++w) ahead[v] = then(ahead[v], waves[w][cl + v]);
            }
            if (later && !gives_state && sub == L::kSubs - 1) {
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    publish(words + tile * step + cl + v, then(ahead[v], mine[v]));
            }
            gather<L>(a.state_in && srow >= 0 ? a.state_in + state : nullptr, some, words, step,
                      tile, items);
        }
        __syncthreads();
        if (part) {
            pack<T, VEC> out[S];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float h = after(ahead[v], start_of<L>(tile, cl + v, items));
                if (later && gives_state && sub == L::kSubs - 1)
                    publish(words + tile * step + cl + v, {0.0f, after(mine[v], h)});
                h = after(before[v], h);
                if (a.saved && t % kSavedSteps == 0 && t < s.n && v < some)
                    a.saved[(static_cast<long long>(b) * ((s.n + kSavedSteps - 1) / kSavedSteps) +
                             t / kSavedSteps) * s.channels + c + v] = h;
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    h = fmaf(f[k][v], h, u[k][v]);
                    out[k][v] = from_float<T>(h);
                }
                if (a.state_out && srow >= 0 && v < some &&
                    (len > 0 ? t < len && len <= t + S : sub == 0 && tile == 0))
                    a.state_out[state + v] = h;
            }
            store_steps<T, L>(y, at_y, s.y_stride, out, full, inside, rows, some);
        } else {
            const pack<T, VEC> out[S] = {};
            store_steps<T, L>(y, at_y, s.y_stride, out, false, 0, rows, some);
        }
        ticket = chained ? next : ticket + gridDim.x;
    }
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes, 4) void scan_last_backward(ScanShape s, ScanBackward a,
                                                                   Chain chain) {
    constexpr int VEC = L::VEC, S = L::S, TL = 64 / L::CL;
    static_assert(L::kSteps % kSavedSteps == 0, "a tile starts from a saved state");
    __shared__ Span waves[L::W][L::kChannels], back[L::W][L::kChannels];
    __shared__ Span items[kGroup][L::kChannels];
    __shared__ unsigned drawn;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int sub = wave * TL + lane / L::CL, cl = lane % L::CL * VEC;
    const auto at_x = lane_offset<L>(s.x_stride), at_gate = lane_offset<L>(s.gate_stride),
               at_y = lane_offset<L>(s.y_stride);
    const bool chained = chain.tiles > 1;
    const int columns = s.batch * chain.slabs;

    unsigned ticket = blockIdx.x;
    if (chained) {
        if (threadIdx.x == 0) drawn = draw(chain);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(drawn);
        __syncthreads();
    }
    while (ticket < chain.total) {
        unsigned next = 0;
        if (chained && threadIdx.x == 0) next = draw(chain);
        const int tile = chain.tiles - 1 - static_cast<int>(ticket / columns);
        const int column = ticket % columns;
        const int b = column / chain.slabs, c0 = column % chain.slabs * L::kChannels, c = c0 + cl;
        const int some = max(0, min(VEC, s.channels - c));
        const int len = length_of(a.lengths, b, s.n);
        const int t0 = tile * L::kSteps, t = t0 + sub * S;
        const int rows = max(0, min(S, s.n - t)), inside = max(0, min(S, len - t));
        const long long row = static_cast<long long>(b) * s.n + t0 + wave * TL * S;  // the wave's first
        T* dx = static_cast<T*>(a.dx) + row * s.x_stride + c0;
        T* dgate = static_cast<T*>(a.dgate) + row * s.gate_stride + c0;
        const bool full = t0 + L::kSteps <= len && c0 + L::kChannels <= s.channels;
        const bool part = t0 < len || tile == 0;
        pack<T, VEC> x[S], g[S], dy[S];
        float f[S][VEC], enter[S][VEC], q[S][VEC];
        Span mine[VEC], before[VEC], behind[VEC], past[VEC];
        if (part) {
            load_steps<T, L>(g, static_cast<const T*>(a.gate) + row * s.gate_stride + c0, at_gate, s.gate_stride,
                             full, inside, some, open_gate<T>());
            load_steps<T, L>(x, static_cast<const T*>(a.x) + row * s.x_stride + c0, at_x, s.x_stride,
                             full, inside, some, static_cast<T>(0.0f));
            load_steps<T, L>(dy, static_cast<const T*>(a.dy) + row * s.y_stride + c0, at_y, s.y_stride,
                             full, inside, some, static_cast<T>(0.0f));
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                mine[v] = {1.0f, 0.0f};
                behind[v] = {1.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    const Gate p = gate_of(to_float<T>(g[k][v]));
                    f[k][v] = p.keep;
                    enter[k][v] = p.enter;
                    mine[v] = then(mine[v], {p.keep, p.enter * to_float<T>(x[k][v])});
                }
#pragma unroll
                for (int k = S - 1; k >= 0; --k)
                    behind[v] = then(behind[v], {f[k][v], f[k][v] * to_float<T>(dy[k][v])});
                before[v] = join_lanes<L::CL, false>(mine[v]);
                past[v] = join_lanes<L::CL, true>(behind[v]);
                if (lane / L::CL == TL - 1) waves[wave][cl + v] = mine[v];
                if (lane / L::CL == 0) back[wave][cl + v] = behind[v];
            }
        }
        if (chained && threadIdx.x == 0) drawn = next;
        __syncthreads();
        if (chained) next = __builtin_amdgcn_readfirstlane(drawn);
        const int last = max(len - 1, 0) / L::kSteps, r = last - tile;
        Word* words = chain.words + static_cast<long long>(column) * L::kChannels;
        const long long step = static_cast<long long>(columns) * L::kChannels;
        const bool gives_state = r % kGroup == 0;
        const bool later = chained && tile > 0;
        const long long state = static_cast<long long>(b) * s.channels + c;
        Span ahead[VEC], rest[VEC];  // of the waves before this one, and of those behind it
        if (part) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ahead[v] = {1.0f, 0.0f};
                rest[v] = {1.0f, 0.0f};
                for (int w = L::W - 1; w > wave; --w) rest[v] = then(rest[v], back[w][cl + v]);
            }
            if (later && !gives_state && sub == 0) {
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    publish(words + r * step + cl + v, then(rest[v], behind[v]));
            }
            gather<L>(a.dstate_out ? a.dstate_out + state : nullptr, some, words, step, r, items);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                for (int w = 0; w < wave; ++w) ahead[v] = then(ahead[v], waves[w][cl + v]);
                float h = 0.0f;
                if (t0 < s.n && v < some)
                    h = a.saved[(static_cast<long long>(b) * ((s.n + kSavedSteps - 1) / kSavedSteps) +
                                 t0 / kSavedSteps) * s.channels + c + v];
                h = after(before[v], after(ahead[v], h));
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    const float in = to_float<T>(x[k][v]);
                    q[k][v] = (h - in) * (f[k][v] * enter[k][v]);
                    h = fmaf(f[k][v], h, enter[k][v] * in);
                }
            }
        }
        __syncthreads();
        if (part) {
            pack<T, VEC> outx[S], outg[S];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                // What reaches this wave's last step from behind it.
                float grad = after(rest[v], start_of<L>(r, cl + v, items));
                if (later && gives_state && sub == 0)
                    publish(words + r * step + cl + v, {0.0f, after(behind[v], grad)});
                grad = after(past[v], grad);
#pragma unroll
                for (int k = S - 1; k >= 0; --k) {
                    const float lam = to_float<T>(dy[k][v]) + grad;
                    outx[k][v] = from_float<T>(enter[k][v] * lam);
                    outg[k][v] = from_float<T>(q[k][v] * lam);
                    grad = f[k][v] * lam;
                }
                if (a.dstate_in && tile == 0 && sub == 0 && v < some) a.dstate_in[state + v] = grad;
            }
            store_steps<T, L>(dx, at_x, s.x_stride, outx, full, inside, rows, some);
            store_steps<T, L>(dgate, at_gate, s.gate_stride, outg, full, inside, rows, some);
        } else {
            const pack<T, VEC> out[S] = {};
            store_steps<T, L>(dx, at_x, s.x_stride, out, false, 0, rows, some);
            store_steps<T, L>(dgate, at_gate, s.gate_stride, out, false, 0, rows, some);
        }
        ticket = chained ? next : ticket + gridDim.x;
    }
}

}  // namespace thff
