// scan_first.hpp -- the gated recurrence on [batch][channels][n] values (the convolutions'
// layout): one pass over the data.  A lane takes 8 or 16 neighbouring steps and composes them; the
// lanes of a row join theirs in registers, its waves through LDS, and where a row takes several
// workgroups, they join through the chain.  Short rows lie side by side in a wave.
//
// Memory bounds it: half 256 x 64 x 4096 takes 70 us (403 MB, 5.7 TB/s; a row is a workgroup's, so
// that nothing waits for another).  float 33 x 96 x 512, a wave a row and all of it in the
// caches: 5.3 us forward and 7.0 backward, the latency of one round of loads, sums and stores.
#pragma once

#include "scan_chain.hpp"

namespace thff {

// V steps a lane, LPR lanes of each of WPR waves a row; a row's tile is kSteps steps.  Chained:
// rows of several tiles, each a workgroup's.  (A kernel for rows of one tile has no code for
// more, which costs registers.)
template <int V_, int LPR_, int WPR_, bool Chained_ = false>
struct Line {
    static constexpr int V = V_, LPR = LPR_, WPR = WPR_, W = WPR_ > 4 ? 8 : 4, kLanes = 64 * W;
    static constexpr int kSteps = LPR * WPR * V, kRows = W / WPR * (64 / LPR);
    static constexpr bool kChained = Chained_;
    static_assert(!kChained || WPR == W, "a workgroup of a chain has one row");
};

// `v` of the lane that Control moves here, `none` where there is none.
template <int Control, int Rows>
__device__ __forceinline__ float moved(float v, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), Control,
                                                      Rows, 0xf, false));
}

template <int Control, int Rows = 0xf>
__device__ __forceinline__ Span moved(Span s) {
    return {moved<Control, Rows>(s.a, 1.0f), moved<Control, Rows>(s.b, 0.0f)};
}

// Joins the spans of groups of LPR lanes: `mine` becomes that of all up to and with this lane,
// the result is that of all before it.
template <int LPR>
__device__ __forceinline__ Span join_line(Span& mine) {
    constexpr Span kNone = {1.0f, 0.0f};
    const int lane = threadIdx.x % LPR;
    static_assert(LPR >= 4 && LPR <= 64 && (LPR & (LPR - 1)) == 0, "a power of two");
    if constexpr (LPR < 16) {
        // Groups that a row of 16 lanes has several of.
        const Span one = moved<0x111>(mine);  // from the lane before
        mine = then(lane >= 1 ? one : kNone, mine);
        const Span two = moved<0x112>(mine);
        mine = then(lane >= 2 ? two : kNone, mine);
        if constexpr (LPR == 8) {
            const Span four = moved<0x114>(mine);
            mine = then(lane >= 4 ? four : kNone, mine);
        }
    } else {
        mine = then(moved<0x111>(mine), mine);
        mine = then(moved<0x112>(mine), mine);
        mine = then(moved<0x114>(mine), mine);
        mine = then(moved<0x118>(mine), mine);
        // A row of 16's last lane to the next row; lane 31 to the upper half.
        if constexpr (LPR >= 32) mine = then(moved<0x142, 0xa>(mine), mine);
        if constexpr (LPR == 64) mine = then(moved<0x143, 0xc>(mine), mine);
    }
    const Span before = moved<0x138>(mine);  // from the lane before, across rows of 16 too
    return lane == 0 ? kNone : before;
}

// The same from the last lane to the first.
template <int LPR>
__device__ __forceinline__ Span join_line_back(Span& mine) {
    const auto mirrored = [](Span s) -> Span { return {__shfl_xor(s.a, LPR - 1), __shfl_xor(s.b, LPR - 1)}; };
    Span m = mirrored(mine);
    const Span before = mirrored(join_line<LPR>(m));
    mine = mirrored(m);
    return before;
}

// A lane's V steps: those of its own that are `in` the sequence; the first `skip` of the vector
// it reads are another lane's (the row ends inside its own).
template <class L>
struct Stretch {
    int row, b, c, tile, len, first, at, skip;
    bool active;

    __device__ __forceinline__ Stretch(const ScanShape& s, const int* lengths, const Chain& chain, int tile_)
        : tile(tile_) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const int rows = s.batch * s.channels;
        const int mine = L::kChained ? chain.column()
                                     : static_cast<int>(chain.block()) * L::kRows +
                                           wave / L::WPR * (64 / L::LPR) + lane / L::LPR;
        active = mine < rows;
        row = min(mine, rows - 1);
        b = chain.by_slabs.quotient(row);
        c = row - b * s.channels;
        len = length_of(lengths, b, s.n);
        first = tile * L::kSteps + (wave % L::WPR * L::LPR + lane % L::LPR) * L::V;
        at = max(0, min(first, s.n - L::V));
        skip = min(first - at, L::V);
    }
    // Whether step i of the vector is the lane's and in the sequence.
    __device__ __forceinline__ bool in(int i) const { return i >= skip && at + i < len; }
    // Whether all of the wave's are.
    __device__ __forceinline__ bool full() const {
        return __ballot(skip == 0 && first + L::V <= len) == ~0ull;
    }
};

// Nothing is read that is not used, but for what a vector reads of another lane's steps.
template <class T, class L>
__device__ __forceinline__ pack<T, L::V> load_line(const T* row, const Stretch<L>& p, int n) {
    if (p.first >= p.len) return pack<T, L::V>{};
    if (n >= L::V) return load_pack<T, L::V>(row + p.at);
    pack<T, L::V> v = {};
#pragma unroll
    for (int i = 0; i < L::V; ++i)
        if (i < n) v[i] = row[i];
    return v;
}

// Stores the lane's steps, zeros past the sequence's end.
template <class T, class L>
__device__ __forceinline__ void store_line(T* row, pack<T, L::V> v, const Stretch<L>& p, int n, bool full) {
    if (!full) {
#pragma unroll
        for (int i = 0; i < L::V; ++i)
            if (!p.in(i)) v[i] = static_cast<T>(0.0f);
    }
    if (!p.active) return;
    if (p.skip == 0 && n >= L::V) {
        store_pack<T, L::V>(row + p.at, v);
    } else {
#pragma unroll
        for (int i = 0; i < L::V; ++i)
            if (i >= p.skip && i < n) row[p.at + i] = v[i];
    }
}

// The chain's link of a row's r-th tile, by the 16 first lanes of a wave, a word each: the
// published state on lane 0, spans of 8 tiles on the next, single ones from lane 8 on.
struct RowLink {
    Word* words;
    long long step;
    int r;
    const Word* at;
    Word word;
    bool has;

    // Asks without waiting.
    __device__ __forceinline__ RowLink(Word* words_, long long step_, int r_) : words(words_), step(step_), r(r_) {
        const int lane = threadIdx.x % 64;
        const int base = (r - 1) / kSuper * kSuper, groups = (r - 1 - base) / kGroup;
        const int single = (r - 1 - base) % kGroup;
        static_assert(kGroup == 8 && kSuper == 64, "at most 7 words of either kind");
        const int tile = lane < 8 ? base + lane * kGroup : base + groups * kGroup + 1 + lane - 8;
        has = r > 0 && (lane < 8 ? lane <= groups : lane - 8 < single);
        at = words + tile * step;
        if (has) word = look(at);
    }

    // Publishes what the tiles behind it need (if `later`) of the tile, whose span is `own`,
    // waits for the answers, and returns the state that the tile starts from, which for r = 0
    // is the one given; all on every lane.
    __device__ __forceinline__ float join(Span own, bool later, float given) {
        constexpr Span kNone = {1.0f, 0.0f};
        const int lane = threadIdx.x % 64;
        const bool publisher = later && lane == 0;
        if (publisher && r % kGroup != 0) publish(words + r * step, own);
        Span mine = kNone;
        if (has) mine = seen(word, at);
        if (r == 0 && lane == 0) mine = {0.0f, given};
        Span near = lane >= 8 ? mine : kNone;
        join_line<16>(near);
        near = {__shfl(near.a, 15), __shfl(near.b, 15)};
        if (publisher && r % kGroup == 0 && r % kSuper != 0) publish(words + r * step, then(near, own));
        join_line<16>(mine);
        const float h = __shfl(mine.b, 15);
        if (publisher && r % kSuper == 0) publish(words + r * step, {0.0f, after(own, h)});
        return h;
    }
};

// Joins a workgroup's waves, whose spans are in `waves` in the order of the chain, and the
// tiles; returns the state before the wave's first step in that order.  `given`: the row's
// first state, on every lane.  own: the wave's place in its row.  Every tile has its place in the
// chain, also past the sequence's end, so that no wait depends on the lengths.
template <class L>
__device__ __forceinline__ float join_tile(const Chain& chain, const Span* waves, float* start, int own,
                                           int r, float given) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if constexpr (L::WPR == 1) return given;
    if constexpr (L::kChained) {
        if (wave == 0) {
            RowLink link(chain.words + chain.column(), chain.columns, r);
            __syncthreads();
            Span all = waves[0];
#pragma unroll
            for (int w = 1; w < L::W; ++w) all = then(all, waves[w]);
            const float h = link.join(all, r + 1 < chain.tiles, given);
            if (threadIdx.x == 0) start[0] = h;
            __syncthreads();
        } else {
            __syncthreads();
            __syncthreads();
        }
        given = start[0];
    } else {
        __syncthreads();
        given = start[wave / L::WPR];
    }
    const Span* before = waves + wave / L::WPR * L::WPR;
    for (int w = 0; w < own; ++w) given = after(before[w], given);
    return given;
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes) void scan_first_forward(ScanShape s, ScanForward a, Chain chain) {
    constexpr int V = L::V;
    __shared__ Span waves[L::W];
    __shared__ float start[L::W];
    __shared__ int drawn;
    if (chain.block() >= chain.blocks) return;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Stretch<L> p(s, a.lengths, chain, L::kChained ? draw_tile(chain, &drawn, 0) : 0);
    const int srow = state_row(s, a.slots, p.b);
    const long long state = static_cast<long long>(srow) * s.channels + p.c;
    pack<T, V> g = {}, x = {};
    if (s.n > 0) {
        g = load_line<T, L>(static_cast<const T*>(a.gate) + p.row * s.gate_stride, p, s.n);
        x = load_line<T, L>(static_cast<const T*>(a.x) + p.row * s.x_stride, p, s.n);
    }
    float given = p.tile == 0 && a.state_in && srow >= 0 ? a.state_in[state] : 0.0f;
    const bool full = p.full();
    float f[V], u[V];
    Span mine = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const Gate q = gate_of(to_float<T>(g[i]));
        f[i] = q.keep;
        u[i] = q.enter * to_float<T>(x[i]);
    }
    if (!full) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!p.in(i)) f[i] = 1.0f, u[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) mine = then_step(mine, f[i], u[i]);
    const Span before = join_line<L::LPR>(mine);
    if (L::WPR > 1) {
        if (lane == 63) waves[wave] = mine;
        // Through LDS, so that it has been read before anyone stores a last state there.
        if (lane == 0 && wave % L::WPR == 0) start[wave / L::WPR] = given;
    }
    float h = join_tile<L>(chain, waves, start, wave % L::WPR, p.tile, given);
    // (No steps save nothing: d_saved has no bytes then, wherever it points.)
    if (a.saved && s.n > 0 && p.active && p.first == p.tile * L::kSteps)
        a.saved[static_cast<long long>(p.row) * chain.tiles + p.tile] = h;
    h = after(before, h);
    pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h = fmaf(f[i], h, u[i]);
        out[i] = from_float<T>(h);
    }
    store_line<T, L>(static_cast<T*>(a.y) + p.row * s.y_stride, out, p, s.n, full);
    // The lane that has the last step, or none to do.
    if (a.state_out && p.active && srow >= 0 &&
        (p.len > 0 ? p.first < p.len && p.len <= p.first + V : p.first == 0))
        a.state_out[state] = h;
}

template <class T, class L>
__global__ __launch_bounds__(L::kLanes) void scan_first_backward(ScanShape s, ScanBackward a, Chain chain) {
    constexpr int V = L::V;
    // Spans of h, and of the gradient that goes back (the last wave's first).
    __shared__ Span waves[L::W], back[L::W];
    __shared__ float start[L::W];
    __shared__ int drawn;
    if (chain.block() >= chain.blocks) return;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Stretch<L> p(s, a.lengths, chain, L::kChained ? chain.tiles - 1 - draw_tile(chain, &drawn, 0) : 0);
    const int r = chain.tiles - 1 - p.tile;
    pack<T, V> g = {}, x = {}, dy = {};
    if (s.n > 0) {
        g = load_line<T, L>(static_cast<const T*>(a.gate) + p.row * s.gate_stride, p, s.n);
        x = load_line<T, L>(static_cast<const T*>(a.x) + p.row * s.x_stride, p, s.n);
        dy = load_line<T, L>(static_cast<const T*>(a.dy) + p.row * s.y_stride, p, s.n);
    }
    float given = r == 0 && a.dstate_out ? a.dstate_out[p.row] : 0.0f;
    float h = s.n > 0 ? a.saved[static_cast<long long>(p.row) * chain.tiles + p.tile] : 0.0f;
    const bool full = p.full();
    float f[V], enter[V], q[V], d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const Gate e = gate_of(to_float<T>(g[i]));
        f[i] = e.keep;
        enter[i] = e.enter;
        q[i] = to_float<T>(x[i]);
        d[i] = to_float<T>(dy[i]);
    }
    if (!full) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!p.in(i)) f[i] = 1.0f, enter[i] = 0.0f, q[i] = 0.0f, d[i] = 0.0f;
    }
    Span mine = {1.0f, 0.0f}, behind = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < V; ++i) mine = then_step(mine, f[i], enter[i] * q[i]);
#pragma unroll
    for (int i = V - 1; i >= 0; --i) behind = then_step(behind, f[i], f[i] * d[i]);
    const Span before = join_line<L::LPR>(mine);
    const Span past = join_line_back<L::LPR>(behind);
    const int own = wave % L::WPR;
    if (L::WPR > 1) {
        if (lane == 63) waves[wave] = mine;
        if (lane == 0) back[wave - own + L::WPR - 1 - own] = behind;
        if (lane == 0 && own == 0) start[wave / L::WPR] = given;
    }
    float grad = join_tile<L>(chain, back, start, L::WPR - 1 - own, r, given);
    for (int w = 0; w < own; ++w) h = after(waves[wave - own + w], h);
    h = after(before, h);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float in = q[i];
        q[i] = (h - in) * (f[i] * enter[i]);
        h = fmaf(f[i], h, enter[i] * in);
    }
    grad = after(past, grad);
    pack<T, V> outx, outg;
#pragma unroll
    for (int i = V - 1; i >= 0; --i) {
        const float lam = d[i] + grad;
        outx[i] = from_float<T>(enter[i] * lam);
        outg[i] = from_float<T>(q[i] * lam);
        grad = f[i] * lam;
    }
    store_line<T, L>(static_cast<T*>(a.dx) + p.row * s.x_stride, outx, p, s.n, full);
    store_line<T, L>(static_cast<T*>(a.dgate) + p.row * s.gate_stride, outg, p, s.n, full);
    if (a.dstate_in && p.active && p.first == 0) a.dstate_in[p.row] = grad;
}

}  // namespace thff
