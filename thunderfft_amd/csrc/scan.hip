// scan.hip -- the gated linear recurrence: per channel, with f = sigmoid(gate),
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  y[t] = h[t],
// and its gradients: lam[t] = dy[t] + f[t+1] lam[t+1],
//   dx[t] = (1 - f[t]) lam[t],  dgate[t] = lam[t] (h[t-1] - x[t]) f[t] (1 - f[t]).
// Values of steps at or past a sequence's length reach no result.
#include <algorithm>

#include "scan_first.hpp"
#include "scan_last.hpp"
#include "scan_step.hpp"

namespace thff {
namespace {

constexpr int kLanes = 256;

// Sets the counters of a chain to zero and empties its words.  (A kernel: a captured memset
// is not replayed reliably.)  Two to five microseconds of a call, its launch most of them: 1 MB
// of words takes 2.0 us, 4.9 MB 4 to 5 (as many with 256 or 1024 workgroups that loop).
__global__ __launch_bounds__(kLanes) void clear_chain(uint4* to, long long counters,
                                                      long long count) {
    for (long long i = static_cast<long long>(blockIdx.x) * kLanes + threadIdx.x; i < count;
         i += static_cast<long long>(gridDim.x) * kLanes) {
        const unsigned v = i < counters ? 0u : ~0u;
        to[i] = make_uint4(v, v, v, v);
    }
}

// Channels last: calls f with the tile type of a shape's forward or backward pass: 4 bytes a
// lane and row.  Lanes along the channels are all 64 of a wave, or 16
//  - where that leaves far fewer of them idle (half 128 x 1000 x 64: 18.7 against 23.5 us forward,
//    37 against 42 backward; 64 x 1000 x 200, which takes 256 or 224: 39 against 26 and 78
//    against 44), and
//  - where one or two columns of tiles are so long that they wait for each other's ends: tiles
//    of four times the steps have a quarter of those (float 1 x 46504 x 64: 21 against 35 and 33
//    against 50 us; half 1 x 65536 x 512, four columns: 83 against 66 and 177 against 117).
template <class T, bool Backward, class F>
auto with_tile(const ScanShape& s, F f) {
    constexpr int VEC = 4 / sizeof(T), S = Backward ? 4 : 8;
    using Wide = Tile<VEC, 64, S, 14, 2, 8>;
    using Thin = Tile<VEC, 16, S, 14, 2, 8>;
    const auto taken = [&](long long channels) {
        return (s.channels + channels - 1) / channels * channels;
    };
    const bool idle = 4 * taken(Wide::kChannels) > 5 * taken(Thin::kChannels);
    const bool long_few = s.batch * taken(Wide::kChannels) <= 2 * Wide::kChannels &&
                          s.n / Wide::kSteps >= kSuper;
    return idle || long_few ? f(Thin{}) : f(Wide{});
}

// Calls f with a value of the shape's type.
template <class F>
auto with_type(const ScanShape& s, F f) {
    if (s.precision == THFF_FLOAT) return f(float{});
    if (s.precision == THFF_HALF) return f(half_t{});
    return f(bfloat_t{});
}

// Rows of more than one tile, both ways; shorter rows have one tile of whatever kind.
using LongLine = Line<8, 64, 8, true>;

// Channels first: calls f with the kind of row for n steps of T: as many lanes as have some, 8
// waves at most.  8 steps a lane; long rows of 2-byte values forward 16 (half 256 x 64 x 4096: 72
// against 79 us; backward, which has more to keep, 123 against 117, and float 117 against 71 at
// 64 x 512 x 1024: its lanes' 64 bytes are four loads that each touch every line).
template <class T, bool Backward, class F>
auto with_line(const ScanShape& s, F f) {
    constexpr int V = !Backward && sizeof(T) == 2 ? 16 : 8;
    const auto within = [&](auto line) { return s.n <= decltype(line)::kSteps; };
    if (within(Line<8, 4, 1>{})) return f(Line<8, 4, 1>{});
    if (within(Line<8, 8, 1>{})) return f(Line<8, 8, 1>{});
    if (within(Line<8, 16, 1>{})) return f(Line<8, 16, 1>{});
    if (within(Line<8, 32, 1>{})) return f(Line<8, 32, 1>{});
    if (within(Line<8, 64, 1>{})) return f(Line<8, 64, 1>{});
    if (within(Line<V, 64, 1>{})) return f(Line<V, 64, 1>{});
    if (within(Line<V, 64, 2>{})) return f(Line<V, 64, 2>{});
    if (within(Line<V, 64, 4>{})) return f(Line<V, 64, 4>{});
    if (within(Line<8, 64, 8>{})) return f(Line<8, 64, 8>{});
    return f(LongLine{});
}

// The chain of a shape whose tiles are `steps` long and `channels` wide (0: one channel, a row).
Chain chain_of(const ScanShape& s, int channels, int steps, void* workspace) {
    Chain chain;
    chain.slabs = channels ? (s.channels + channels - 1) / channels : s.channels;
    chain.tiles = s.n > 0 ? (s.n + steps - 1) / steps : 1;
    chain.columns = static_cast<unsigned>(s.batch) * chain.slabs;
    // (An empty shape has no columns, and launches nothing.)
    chain.by_columns = Divider(std::max(chain.columns, 1u));
    chain.by_slabs = Divider(std::max(chain.slabs, 1));
    chain.drawn = static_cast<unsigned*>(workspace);
    chain.words = reinterpret_cast<Word*>(static_cast<char*>(workspace) +
                                          static_cast<long long>(chain.columns) * kCounterBytes);
    return chain;
}

template <class L>
Chain last_chain(const ScanShape& s, void* workspace) {
    Chain chain = chain_of(s, L::kChannels, L::kSteps, workspace);
    chain.blocks = chain.columns * chain.tiles;
    return chain;
}

template <class L>
Chain first_chain(const ScanShape& s, void* workspace) {
    Chain chain = chain_of(s, 0, L::kSteps, workspace);
    chain.blocks = L::kChained ? chain.columns * chain.tiles
                               : static_cast<unsigned>((chain.columns + static_cast<long long>(L::kRows) - 1) / L::kRows);
    return chain;
}

dim3 grid_of(const Chain& chain) {
    constexpr unsigned kMost = 1u << 21;
    return dim3(std::min(chain.blocks, kMost), (chain.blocks + kMost - 1) / kMost);
}

long long chain_bytes(const Chain& chain, int channels) {
    if (chain.tiles <= 1) return 0;
    const long long words = static_cast<long long>(chain.columns) * std::max(channels, 1) * chain.tiles;
    return (chain.columns * static_cast<long long>(kCounterBytes) + 8 * words + 15) / 16 * 16;
}

// Whether the workgroups of all tiles can be counted.
bool chain_fits(const ScanShape& s, const Chain& chain) {
    return static_cast<__int128>(s.batch) * chain.slabs * chain.tiles <= 0x7fffffff;
}

hipError_t clear(const Chain& chain, int channels, hipStream_t stream) {
    const long long count = chain_bytes(chain, channels) / 16;
    if (count == 0) return hipSuccess;
    const long long blocks = std::min((count + kLanes - 1) / kLanes, 1LL << 20);
    clear_chain<<<static_cast<unsigned>(blocks), kLanes, 0, stream>>>(
        reinterpret_cast<uint4*>(chain.drawn), chain.columns * (kCounterBytes / 16LL), count);
    return hipGetLastError();
}

template <class L, class Args>
hipError_t launch_last(void (*kernel)(ScanShape, Args, Chain), const ScanShape& s, const Args& a,
                       hipStream_t stream) {
    const Chain chain = last_chain<L>(s, a.workspace);
    const hipError_t err = clear(chain, L::kChannels, stream);
    if (err != hipSuccess) return err;
    kernel<<<grid_of(chain), L::kLanes, 0, stream>>>(s, a, chain);
    return hipGetLastError();
}

template <class L, class Args>
hipError_t launch_first(void (*kernel)(ScanShape, Args, Chain), const ScanShape& s, const Args& a,
                        hipStream_t stream) {
    const Chain chain = first_chain<L>(s, a.workspace);
    const hipError_t err = clear(chain, 0, stream);
    if (err != hipSuccess) return err;
    kernel<<<grid_of(chain), L::kLanes, 0, stream>>>(s, a, chain);
    return hipGetLastError();
}

// One step: 16 bytes of states a lane where the channels lie side by side.
template <class T>
hipError_t launch_step(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    const auto channel = [&](long long stride) { return s.channels_first ? stride : 1LL; };
    const auto row = [&](long long stride) { return s.channels_first ? s.channels * stride : stride; };
    const StepStrides d{channel(s.x_stride), channel(s.gate_stride), channel(s.y_stride),
                        row(s.x_stride),     row(s.gate_stride),     row(s.y_stride)};
    const auto launch = [&](void (*kernel)(ScanShape, ScanForward, StepStrides), int channels) {
        const long long lanes = static_cast<long long>(s.batch) * ((s.channels + channels - 1) / channels);
        kernel<<<static_cast<unsigned>((lanes + kStepLanes - 1) / kStepLanes), kStepLanes, 0, stream>>>(s, a, d);
        return hipGetLastError();
    };
    if (d.x == 1 && d.gate == 1 && d.y == 1) return launch(scan_step<T, 4>, 4);
    return launch(scan_step<T, 1>, 1);
}

template <class T>
hipError_t forward_of(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    if (s.n == 1) return launch_step<T>(s, a, stream);
    if (s.channels_first)
        return with_line<T, false>(s, [&](auto line) {
            using L = decltype(line);
            return launch_first<L>(scan_first_forward<T, L>, s, a, stream);
        });
    return with_tile<T, false>(s, [&](auto tile) {
        using L = decltype(tile);
        return launch_last<L>(scan_last_forward<T, L>, s, a, stream);
    });
}

template <class T>
hipError_t backward_of(const ScanShape& s, const ScanBackward& a, hipStream_t stream) {
    if (s.channels_first)
        return with_line<T, true>(s, [&](auto line) {
            using L = decltype(line);
            return launch_first<L>(scan_first_backward<T, L>, s, a, stream);
        });
    return with_tile<T, true>(s, [&](auto tile) {
        using L = decltype(tile);
        return launch_last<L>(scan_last_backward<T, L>, s, a, stream);
    });
}

}  // namespace

long long scan_saved_bytes(const ScanShape& s) {
    if (s.n == 0) return 0;
    const long long rows = static_cast<long long>(s.batch) * s.channels;
    if (s.channels_first) return 4 * rows * first_chain<LongLine>(s, nullptr).tiles;
    return 4 * rows * ((static_cast<long long>(s.n) + kSaved - 1) / kSaved);
}

long long scan_workspace_bytes(const ScanShape& s) {
    if (s.channels_first) return chain_bytes(first_chain<LongLine>(s, nullptr), 0);
    const auto bytes = [&](auto tile) {
        using L = decltype(tile);
        return chain_bytes(last_chain<L>(s, nullptr), L::kChannels);
    };
    return with_type(s, [&](auto v) {
        using T = decltype(v);
        return std::max(with_tile<T, false>(s, bytes), with_tile<T, true>(s, bytes));
    });
}

bool scan_fits(const ScanShape& s) {
    if (static_cast<long long>(s.batch) * s.channels > 0x7fffff00LL) return false;
    if (s.channels_first) return chain_fits(s, first_chain<LongLine>(s, nullptr));
    const auto fits = [&](auto tile) { return chain_fits(s, last_chain<decltype(tile)>(s, nullptr)); };
    return with_type(s, [&](auto v) {
        using T = decltype(v);
        return with_tile<T, false>(s, fits) && with_tile<T, true>(s, fits);
    });
}

hipError_t launch_gated_scan(const ScanShape& s, const ScanForward& a, hipStream_t stream) {
    return with_type(s, [&](auto v) { return forward_of<decltype(v)>(s, a, stream); });
}

hipError_t launch_gated_scan_backward(const ScanShape& s, const ScanBackward& a,
                                      hipStream_t stream) {
    return with_type(s, [&](auto v) { return backward_of<decltype(v)>(s, a, stream); });
}

}  // namespace thff
