// scan_chain.hpp -- what the gated recurrence's kernels of both layouts share: gates, spans of
// steps, and the chain that joins the tiles of a long axis.
//
// A step is h -> f h + u with u = (1 - f) x.  Steps compose: (A, B) then (f, u) is
// (f A, f B + u).  Workgroups take a tile of steps each; a tile's (A, B) is published for the
// tiles behind it.  Counted from the first, every 64th tile publishes the state after it
// instead, and every 8th the span of the 8 tiles up to it: a tile starts from the last such
// state before it, led through at most 7 spans of 8 tiles and 7 of single ones, always in this
// order, so that the result does not depend on timing.  Only every 64th tile waits for
// another's wait.  The backward pass goes the same way from the last step to the first, with
// c -> f (dy + c), c the gradient that reaches a step from the steps behind it.
//
// Published words are 64 bits, (A, B) or (0, state), and empty ones all ones: each is valid as
// soon as it is seen, without fences.  A workgroup draws its tile from a counter of its column,
// first steps first, publishes before it waits, and waits only for tiles drawn earlier, which
// running workgroups hold: every wait ends.  (One counter for all columns takes 11.6 ns a draw,
// 48 us for 4096 workgroups; one for each takes nothing.)
//
// A workgroup takes one tile and ends: one that goes on to the next waits, with the first load
// it needs, for its last tile's stores, which the same counter counts.
#pragma once

#include "sequence.hpp"
#include "sequence_io.hpp"

namespace thff {

struct Gate {
    float keep;   // sigmoid(g)
    float enter;  // 1 - sigmoid(g) = sigmoid(-g)
};

// Both from e = exp(-g), so that neither cancels; e is held at 2^126, where f is 2^-126 and
// 1 - f is 1, so that it does not overflow.  A NaN stays one (the minimum that keeps it).
__device__ __forceinline__ Gate gate_of(float g) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(-1.44269504f * g, 126.0f));
    const float f = __builtin_amdgcn_rcpf(1.0f + e);
    return {f, e * f};
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

constexpr int kGroup = 8, kSuper = 64;

// (A, B) of some steps: h -> A h + B.
struct Span {
    float a, b;
};

// An infinite state stays infinite: each gate is above zero, also where their product has been
// rounded to zero.  A finite state takes the product as it is: below 2^-126 it has fewer bits, and
// what is left of the state is off by 2^-150 of it for each joining.  (A product held at 2^-149 for
// all states leaves 1.4e-7 of 1e38 for good.  The choice costs 0.5% of bfloat16 8 x 4096 x 2048
// forward, 89.9 us with the chain's clearing, and 1.5% of 16 x 64 x 65536, channels first, 87.0 us.)
__device__ __forceinline__ float after(Span s, float h) {
    return fmaf(__builtin_isinf(h) ? 1.0f : s.a, h, s.b);
}

__device__ __forceinline__ Span then(Span first, Span second) {
    return {first.a * second.a, after(second, first.b)};
}

// One step more.
__device__ __forceinline__ Span then_step(Span first, float f, float u) {
    return {first.a * f, fmaf(f, first.b, u)};
}

using Word = unsigned long long;

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

// Division by a number that the host knows: n / d = n m >> shift for n < 2^31, with
// 2^(s-1) < d <= 2^s, shift = 31 + s and m = ceil(2^shift / d), which is off by less than d
// units of 2^-shift a unit of n: too little to reach the next whole number.
struct Divider {
    unsigned d, m;
    int shift;

    Divider() = default;
    explicit Divider(unsigned by) : d(by), shift(31) {
        while ((1ull << (shift - 31)) < by) ++shift;
        m = static_cast<unsigned>(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ int quotient(unsigned n) const {
        return static_cast<int>(static_cast<unsigned long long>(n) * m >> shift);
    }
};

// The workspace: a counter for every column of tiles, far enough apart, then a word for every
// channel of every tile.
struct Chain {
    unsigned* drawn;
    Word* words;
    int slabs, tiles;  // tiles along the channels, along the steps
    unsigned columns;  // batch * slabs
    unsigned blocks;   // workgroups
    Divider by_columns, by_slabs;

    // A launch has less than 2^32 lanes along x, so many workgroups take rows of a grid.
    __device__ __forceinline__ unsigned block() const { return blockIdx.y * gridDim.x + blockIdx.x; }
    // The column of a workgroup, and the tile of it that it expects to draw.
    __device__ __forceinline__ int expected() const { return by_columns.quotient(block()); }
    __device__ __forceinline__ int column() const { return block() - expected() * columns; }
};
constexpr int kCounterBytes = 64;

// What a tile publishes for a channel.
__device__ __forceinline__ Span seen(Word& w, const Word* at) {
    while (static_cast<unsigned>(w) == ~0u) w = look(at);
    return span_of(w);
}

// N channels of the r-th tile of a chain.  words: theirs of the chain's first tile; step:
// words from a tile to the next.
template <int N>
struct Link {
    Word* words;
    long long step;
    int r;
    Word one[kGroup - 1][N], group[kSuper / kGroup - 1][N], state[N];

    __device__ __forceinline__ int base() const { return (r - 1) / kSuper * kSuper; }
    __device__ __forceinline__ int groups() const { return (r - 1 - base()) / kGroup; }
    __device__ __forceinline__ int single() const { return (r - 1 - base()) % kGroup; }
    __device__ __forceinline__ const Word* at_one(int i) const {
        return words + (base() + groups() * kGroup + 1 + i) * step;
    }
    __device__ __forceinline__ const Word* at_group(int i) const {
        return words + (base() + (i + 1) * kGroup) * step;
    }

    // Asks for what the tile needs of those before it, without waiting.
    __device__ __forceinline__ void ask() {
        if (r == 0) return;
#pragma unroll
        for (int i = 0; i < kGroup - 1; ++i)
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (i < single()) one[i][v] = look(at_one(i) + v);
#pragma unroll
        for (int i = 0; i < kSuper / kGroup - 1; ++i)
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (i < groups()) group[i][v] = look(at_group(i) + v);
#pragma unroll
        for (int v = 0; v < N; ++v) state[v] = look(words + base() * step + v);
    }

    // Publishes what the tiles behind it need (if `later`) of the tile, whose span is `own`,
    // waits for the answers, and returns the state that the tile starts from, which for
    // r = 0 is the one given.
    __device__ __forceinline__ void join(float (&h)[N], const Span (&own)[N], bool later,
                                         const float (&given)[N]) {
        Word* here = words + r * step;
        if (later && r % kGroup != 0) {
#pragma unroll
            for (int v = 0; v < N; ++v) publish(here + v, own[v]);
        }
#pragma unroll
        for (int v = 0; v < N; ++v) h[v] = given[v];
        if (r > 0) {
            Span near[N];
#pragma unroll
            for (int v = 0; v < N; ++v) near[v] = {1.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kGroup - 1; ++i)
#pragma unroll
                for (int v = 0; v < N; ++v)
                    if (i < single()) near[v] = then(near[v], seen(one[i][v], at_one(i) + v));
            if (later && r % kGroup == 0 && r % kSuper != 0) {
#pragma unroll
                for (int v = 0; v < N; ++v) publish(here + v, then(near[v], own[v]));
            }
#pragma unroll
            for (int v = 0; v < N; ++v) h[v] = seen(state[v], words + base() * step + v).b;
#pragma unroll
            for (int i = 0; i < kSuper / kGroup - 1; ++i)
#pragma unroll
                for (int v = 0; v < N; ++v)
                    if (i < groups()) h[v] = after(seen(group[i][v], at_group(i) + v), h[v]);
#pragma unroll
            for (int v = 0; v < N; ++v) h[v] = after(near[v], h[v]);
        }
        if (later && r % kSuper == 0) {
#pragma unroll
            for (int v = 0; v < N; ++v) publish(here + v, {0.0f, after(own[v], h[v])});
        }
    }
};

template <class T>
__device__ __forceinline__ T open_gate() {
    return static_cast<T>(__builtin_inff());
}

// Draws the workgroup's tile of its column, by the first lane of wave `drawer`.
__device__ __forceinline__ int draw_tile(const Chain& chain, int* drawn, int drawer) {
    if (static_cast<int>(threadIdx.x) == 64 * drawer) {
        unsigned* counter = chain.drawn + chain.column() * (kCounterBytes / 4LL);
        *drawn = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*drawn);
}

}  // namespace thff
