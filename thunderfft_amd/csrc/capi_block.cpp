// capi_block.cpp -- the C ABI of a state space block's operators of
// include/thunderfft/thunderfft.h: argument checks, all before any HIP call, and dispatch.
#include <hip/hip_runtime.h>

#include <initializer_list>
#include <string>

#include "block.hpp"
#include "capi_checks.hpp"
#include "state_cut.hpp"

namespace {

using namespace thff;

constexpr long long kMostChannels = 0x7fffff00LL;  // batch * channels

bool all_aligned(std::initializer_list<const void*> pointers, unsigned bytes) {
    for (const void* p : pointers)
        if (!aligned(p, bytes)) return false;
    return true;
}

bool any_null(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (!p) return true;
    return false;
}

// Whether an output is an input or another output (null pointers are none).  Arrays of no bytes are given
// as null: they may lie where another begins.
bool any_alias(std::initializer_list<const void*> outputs, std::initializer_list<const void*> inputs) {
    for (const void* const* o = outputs.begin(); o != outputs.end(); ++o) {
        if (!*o) continue;
        for (const void* i : inputs)
            if (i == *o) return true;
        for (const void* const* other = o + 1; other != outputs.end(); ++other)
            if (*other == *o) return true;
    }
    return false;
}

int check_sizes(const char* who, int precision, int batch, int n, int channels) {
    if (!value_type(precision))
        return fail(THFF_EINVAL, std::string(who) + " supports float, half and bfloat16 only");
    if (batch < 0 || n < 0 || channels < 0)
        return fail(THFF_EINVAL, std::string(who) + " batch, n and channels must be nonnegative");
    if (batch > kMostSize || n > kMostSize || channels > kMostSize)
        return fail(THFF_EINVAL, std::string(who) + " batch, n and channels must be at most 2^30");
    if (static_cast<long long>(batch) * channels > kMostChannels)
        return fail(THFF_EINVAL, std::string(who) + " batch * channels must be at most 2^31 - 256");
    return THFF_OK;
}

int check_shape(const thff_conv_shape* shape, ConvShape* out) {
    if (!shape) return fail(THFF_EINVAL, "thff_conv_shape is null");
    const int rc = check_sizes("ThunderFFT_short_conv", shape->precision, shape->batch, shape->n, shape->channels);
    if (rc != THFF_OK) return rc;
    if (shape->width < 2 || shape->width > 4)
        return fail(THFF_EINVAL, "ThunderFFT_short_conv width must be 2 to 4");
    if (shape->silu != 0 && shape->silu != 1)
        return fail(THFF_EINVAL, "ThunderFFT_short_conv silu must be 0 or 1");
    *out = ConvShape{shape->precision, shape->silu == 1, shape->batch, shape->n, shape->channels,
                     shape->width,     shape->states,    0,            0};
    const long long rows = static_cast<long long>(shape->batch) * shape->n;
    if (!stride_of(shape->x_stride, shape->channels, rows, &out->x_stride) ||
        !stride_of(shape->y_stride, shape->channels, rows, &out->y_stride))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv stride is shorter than a row or too long");
    return THFF_OK;
}

int conv_impl(const thff_conv_shape* shape, const ConvForward& a, void* stream, bool synchronize) {
    ConvShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (s.batch == 0 || s.channels == 0) return THFF_OK;
    const unsigned e = element_bytes(s.precision);
    if (!a.weight || (s.n > 0 && any_null({a.x, a.y})))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv requires non-null x, weight and y");
    const bool steps = s.n > 0;
    if ((steps && any_alias({a.y}, {a.x, a.weight, a.bias, a.state_in, a.state_out, a.slots, a.lengths})) ||
        any_alias({a.state_out}, {steps ? a.x : nullptr, a.weight, a.bias, a.slots, a.lengths}))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv output must not alias another array");
    if (!all_aligned({a.x, a.y, a.state_in, a.state_out}, e))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv requires element-aligned values and states");
    if (!all_aligned({a.weight, a.bias, a.slots, a.lengths}, 4))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv requires 4-byte aligned weights, slots and lengths");
    if (a.slots && s.states < 0)
        return fail(THFF_EINVAL, "ThunderFFT_short_conv states must be nonnegative");
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_short_conv(s, a, st), st, synchronize, "ThunderFFT_short_conv");
}

int conv_backward_impl(const thff_conv_shape* shape, const ConvBackward& a, void* stream,
                       bool synchronize) {
    ConvShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (s.channels == 0) return THFF_OK;
    const unsigned e = element_bytes(s.precision);
    if (s.batch > 0 && (!a.weight || (s.n > 0 && any_null({a.dy, a.x, a.dx}))))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward requires non-null dy, x, weight and dx");
    if (s.batch > 0 && s.n > 0) {
        if (!a.workspace && (a.dweight || a.dbias) && conv_workspace_bytes(s) > 0)
            return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward requires a workspace of " +
                                         std::to_string(conv_workspace_bytes(s)) + " bytes");
    }
    const bool scratch = (a.dweight || a.dbias) && conv_workspace_bytes(s) > 0;
    const bool steps = s.batch > 0 && s.n > 0;
    if (any_alias({steps ? a.dx : nullptr, a.dweight, a.dbias, a.dstate_in, scratch ? a.workspace : nullptr},
                  {steps ? a.dy : nullptr, steps ? a.x : nullptr, a.weight, a.bias, a.state_in, a.dstate_out, a.lengths}))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward outputs must not alias other arrays");
    if (!all_aligned({a.dy, a.x, a.dx, a.state_in, a.dstate_out, a.dstate_in}, e))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward requires element-aligned values and states");
    if (!all_aligned({a.weight, a.bias, a.dweight, a.dbias, a.lengths}, 4))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward requires 4-byte aligned weights and lengths");
    if (!aligned(a.workspace, 16))
        return fail(THFF_EINVAL, "ThunderFFT_short_conv_backward requires a 16-byte aligned workspace");
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_short_conv_backward(s, a, st), st, synchronize, "ThunderFFT_short_conv_backward");
}

int check_shape(const thff_state_shape* shape, StateShape* out) {
    if (!shape) return fail(THFF_EINVAL, "thff_state_shape is null");
    const int rc = check_sizes("ThunderFFT_state_scan", shape->precision, shape->batch, shape->n, shape->channels);
    if (rc != THFF_OK) return rc;
    if (shape->order < 1 || shape->order > 64)
        return fail(THFF_EINVAL, "ThunderFFT_state_scan order must be 1 to 64");
    if (shape->groups < 1 || shape->channels % shape->groups != 0)
        return fail(THFF_EINVAL, "ThunderFFT_state_scan groups must divide the channels");
    *out = StateShape{shape->precision, shape->batch,  shape->n, shape->channels, shape->order,
                      shape->groups,    shape->states, 0,        0,               0,
                      0,                0,             0};
    const long long rows = static_cast<long long>(shape->batch) * shape->n;
    const long long shared = static_cast<long long>(shape->groups) * shape->order;
    if (!stride_of(shape->x_stride, shape->channels, rows, &out->x_stride) ||
        !stride_of(shape->delta_stride, shape->channels, rows, &out->delta_stride) ||
        !stride_of(shape->gate_stride, shape->channels, rows, &out->gate_stride) ||
        !stride_of(shape->y_stride, shape->channels, rows, &out->y_stride) ||
        !stride_of(shape->b_stride, shared, rows, &out->b_stride) ||
        !stride_of(shape->c_stride, shared, rows, &out->c_stride))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan stride is shorter than a row or too long");
    for (long long stride : {out->x_stride, out->delta_stride, out->gate_stride, out->y_stride, out->b_stride, out->c_stride})
        if (stride > kStateStride) return fail(THFF_EINVAL, "ThunderFFT_state_scan stride must be at most 2^24");
    if (!state_fits(*out)) return fail(THFF_EINVAL, "ThunderFFT_state_scan shape exceeds one launch");
    return THFF_OK;
}

int state_impl(const thff_state_shape* shape, const StateForward& a, void* stream, bool synchronize) {
    StateShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (s.batch == 0 || s.channels == 0) return THFF_OK;
    if (!a.a || (s.n > 0 && any_null({a.x, a.delta, a.b, a.c, a.y})))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan requires non-null x, delta, a, b, c and y");
    const bool steps = s.n > 0;
    if ((steps && any_alias({a.y, a.saved, state_forward_bytes(s) > 0 ? a.workspace : nullptr},
                            {a.x, a.delta, a.a, a.b, a.c, a.skip, a.gate, a.delta_bias, a.state_in, a.state_out, a.slots,
                             a.lengths})) ||
        (steps && any_alias({a.state_out}, {a.x, a.delta, a.b, a.c, a.gate})) ||
        any_alias({a.state_out}, {a.a, a.skip, a.delta_bias, a.slots, a.lengths}))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan output must not alias another array");
    if (!all_aligned({a.x, a.delta, a.b, a.c, a.gate, a.y}, element_bytes(s.precision)))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan requires element-aligned buffers");
    if (!all_aligned({a.a, a.skip, a.delta_bias, a.state_in, a.state_out, a.slots, a.lengths}, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_state_scan requires 4-byte aligned weights, states, slots and lengths");
    if (a.slots && s.states < 0)
        return fail(THFF_EINVAL, "ThunderFFT_state_scan states must be nonnegative");
    if (!all_aligned({a.saved, a.workspace}, 16))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan requires 16-byte aligned saved and workspace");
    if (!a.workspace && state_forward_bytes(s) > 0)
        return fail(THFF_EINVAL, "ThunderFFT_state_scan requires a workspace of " +
                                     std::to_string(state_forward_bytes(s)) + " bytes");
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_state_scan(s, a, st), st, synchronize, "ThunderFFT_state_scan");
}

int state_backward_impl(const thff_state_shape* shape, const thff_state_gradients* g, void* workspace,
                        void* stream, bool synchronize) {
    StateShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (!g) return fail(THFF_EINVAL, "thff_state_gradients is null");
    if (s.channels == 0) return THFF_OK;
    if (!g->da) return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires non-null da");
    if (s.batch > 0 && (!g->a || (s.n > 0 && any_null({g->dy, g->x, g->delta, g->b, g->c, g->dx, g->ddelta, g->db, g->dc}))))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires non-null dy, x, delta, a, b, c, dx, "
                                 "ddelta, db and dc");
    if (s.batch > 0 && s.n > 0) {
        if (g->gate && !g->dgate)
            return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires dgate where there is a gate");
        if (!g->saved)
            return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires what the forward call saved");
    }
    if (s.batch > 0 && !workspace && state_workspace_bytes(s) > 0)
        return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires a workspace of " +
                                     std::to_string(state_workspace_bytes(s)) + " bytes");
    const void* scratch = state_workspace_bytes(s) > 0 ? workspace : nullptr;
    const bool steps = s.batch > 0 && s.n > 0;
    if ((steps && any_alias({g->dx, g->ddelta, g->db, g->dc, g->dgate},
                            {g->dy, g->x, g->delta, g->a, g->b, g->c, g->skip, g->gate, g->delta_bias, g->saved, g->dstate_out,
                             g->lengths, g->da, g->dskip, g->ddelta_bias, g->dstate_in, scratch})) ||
        (steps && any_alias({g->da, g->dskip, g->ddelta_bias, g->dstate_in, scratch},
                            {g->dy, g->x, g->delta, g->b, g->c, g->gate, g->saved})) ||
        any_alias({g->da, g->dskip, g->ddelta_bias, g->dstate_in, scratch},
                  {g->a, g->skip, g->delta_bias, g->dstate_out, g->lengths}))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward outputs must not alias other arrays");
    if (!all_aligned({g->dy, g->x, g->delta, g->b, g->c, g->gate, g->dx, g->ddelta, g->db, g->dc, g->dgate},
                     element_bytes(s.precision)))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires element-aligned buffers");
    if (!all_aligned({g->a, g->skip, g->delta_bias, g->dstate_out, g->lengths, g->da, g->dskip, g->ddelta_bias,
                      g->dstate_in}, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_state_scan_backward requires 4-byte aligned weights, states and lengths");
    if (!all_aligned({g->saved, workspace}, 16))
        return fail(THFF_EINVAL, "ThunderFFT_state_scan_backward requires 16-byte aligned saved and workspace");
    const StateBackward a{g->dy,
                          g->x,
                          g->delta,
                          static_cast<const float*>(g->a),
                          g->b,
                          g->c,
                          static_cast<const float*>(g->skip),
                          g->gate,
                          static_cast<const float*>(g->delta_bias),
                          static_cast<const float*>(g->saved),
                          static_cast<const float*>(g->dstate_out),
                          static_cast<const int*>(g->lengths),
                          g->dx,
                          g->ddelta,
                          static_cast<float*>(g->da),
                          g->db,
                          g->dc,
                          static_cast<float*>(g->dskip),
                          g->gate ? g->dgate : nullptr,
                          static_cast<float*>(g->ddelta_bias),
                          static_cast<float*>(g->dstate_in),
                          static_cast<float*>(workspace)};
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_state_scan_backward(s, a, st), st, synchronize, "ThunderFFT_state_scan_backward");
}

int check_rms(int precision, long long rows, int cols) {
    if (!value_type(precision))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm supports float, half and bfloat16 only");
    if (rows < 0) return fail(THFF_EINVAL, "ThunderFFT_rms_norm rows must be nonnegative");
    if (cols < 1 || cols > kMostSize)
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm cols must be 1 to 2^30");
    return THFF_OK;
}

// a.block = 0: y is of the type of the values.
int rms_impl(RmsForward a, void* stream, bool synchronize) {
    const int rc = check_rms(a.precision, a.rows, a.cols);
    if (rc != THFF_OK) return rc;
    if (!(a.eps >= 0.0f)) return fail(THFF_EINVAL, "ThunderFFT_rms_norm eps must be nonnegative");
    if (!stride_of(a.x_stride, a.cols, a.rows, &a.x_stride) ||
        !stride_of(a.residual_stride, a.cols, a.rows, &a.residual_stride) ||
        !stride_of(a.y_stride, a.cols, a.rows, &a.y_stride) ||
        !stride_of(a.sum_stride, a.cols, a.rows, &a.sum_stride))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm stride is shorter than a row or too long");
    const bool bits8 = a.block != 0;
    if (bits8 && a.block != 128 && a.block != a.cols)
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm_8bit block must be 128 or cols");
    if (a.rows == 0) return THFF_OK;
    if (!a.x || !a.y) return fail(THFF_EINVAL, "ThunderFFT_rms_norm requires non-null x and output");
    if (bits8 && !a.scales) return fail(THFF_EINVAL, "ThunderFFT_rms_norm_8bit requires non-null scales");
    if (any_alias({a.y, a.sum, a.scales, a.rstd}, {a.x, a.weight}) || any_alias({a.y, a.scales, a.rstd}, {a.residual}))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm outputs must not alias its inputs");
    if (a.sum && a.sum == a.residual && a.sum_stride != a.residual_stride)
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm sums in the residual's place need its stride");
    const unsigned e = element_bytes(a.precision);
    if (!all_aligned({a.x, a.residual, a.sum}, e) || !aligned(a.y, bits8 ? 1 : e))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm requires element-aligned buffers");
    if (!all_aligned({a.weight, a.rstd, a.scales}, 4))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm requires 4-byte aligned weights, scales and statistics");
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_rms_norm(a, st), st, synchronize, "ThunderFFT_rms_norm");
}

int rms_backward_impl(RmsBackward a, void* stream, bool synchronize) {
    const int rc = check_rms(a.precision, a.rows, a.cols);
    if (rc != THFF_OK) return rc;
    if (!stride_of(a.dy_stride, a.cols, a.rows, &a.dy_stride) ||
        !stride_of(a.sum_stride, a.cols, a.rows, &a.sum_stride) ||
        !stride_of(a.dsum_stride, a.cols, a.rows, &a.dsum_stride) ||
        !stride_of(a.dx_stride, a.cols, a.rows, &a.dx_stride))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward stride is shorter than a row or too long");
    if (a.rows == 0 && !a.dweight) return THFF_OK;
    if (a.rows > 0) {
        if (any_null({a.dy, a.sum, a.rstd, a.dx}))
            return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward requires non-null dy, sum, rstd and dx");
        const bool scratch = a.dweight && rms_workspace_bytes(a.rows, a.cols) > 0;
        if (any_alias({a.dx, a.dweight, scratch ? a.workspace : nullptr}, {a.dy, a.sum, a.rstd, a.weight, a.dsum}))
            return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward outputs must not alias its inputs");
        if (!all_aligned({a.dy, a.sum, a.dsum, a.dx}, element_bytes(a.precision)))
            return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward requires element-aligned buffers");
        if (!a.workspace && a.dweight && rms_workspace_bytes(a.rows, a.cols) > 0)
            return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward requires a workspace of " +
                                         std::to_string(rms_workspace_bytes(a.rows, a.cols)) + " bytes");
    }
    if (!all_aligned({a.weight, a.rstd, a.dweight}, 4))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward requires 4-byte aligned weights and statistics");
    if (!aligned(a.workspace, 16))
        return fail(THFF_EINVAL, "ThunderFFT_rms_norm_backward requires a 16-byte aligned workspace");
    auto st = static_cast<hipStream_t>(stream);
    return finish(launch_rms_norm_backward(a, st), st, synchronize, "ThunderFFT_rms_norm_backward");
}

int rms_8bit(const RmsForward& a, void* stream, bool synchronize) {
    // 0 stands for no blocks inside.
    if (a.block == 0) return fail(THFF_EINVAL, "ThunderFFT_rms_norm_8bit block must be 128 or cols");
    return rms_impl(a, stream, synchronize);
}

const float* floats(const void* p) { return static_cast<const float*>(p); }
float* floats(void* p) { return static_cast<float*>(p); }
const int* ints(const void* p) { return static_cast<const int*>(p); }

}  // namespace

extern "C" {

long long thff_short_conv_workspace_bytes(const thff_conv_shape* shape) {
    return guarded([&]() -> long long {
        ConvShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? conv_workspace_bytes(s) : rc;
    });
}

#define THFF_TWINS(name, parameters, call)                            \
    int name parameters {                                             \
        constexpr bool synchronize = true;                            \
        return guarded([&] { return call; });                         \
    }                                                                 \
    int name##_async parameters {                                     \
        constexpr bool synchronize = false;                           \
        return guarded([&] { return call; });                         \
    }

THFF_TWINS(thff_short_conv,
           (const thff_conv_shape* shape, const void* d_x, const void* d_weight, const void* d_bias, void* d_y,
            const void* d_state_in, void* d_state_out, const void* d_slots, const void* d_lengths, void* stream),
           conv_impl(shape,
                     ConvForward{d_x, floats(d_weight), floats(d_bias), d_state_in, ints(d_slots), ints(d_lengths), d_y,
                                 d_state_out},
                     stream, synchronize))

THFF_TWINS(thff_short_conv_backward,
           (const thff_conv_shape* shape, const void* d_dy, const void* d_x, const void* d_weight, const void* d_bias,
            const void* d_state_in, const void* d_dstate_out, const void* d_lengths, void* d_dx, void* d_dweight,
            void* d_dbias, void* d_dstate_in, void* d_workspace, void* stream),
           conv_backward_impl(shape,
                              ConvBackward{d_dy, d_x, floats(d_weight), floats(d_bias), d_state_in, d_dstate_out,
                                           ints(d_lengths), d_dx, floats(d_dweight), floats(d_dbias), d_dstate_in,
                                           floats(d_workspace)},
                              stream, synchronize))

long long thff_state_scan_saved_bytes(const thff_state_shape* shape) {
    return guarded([&]() -> long long {
        StateShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? state_saved_bytes(s) : rc;
    });
}

long long thff_state_scan_forward_bytes(const thff_state_shape* shape) {
    return guarded([&]() -> long long {
        StateShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? state_forward_bytes(s) : rc;
    });
}

long long thff_state_scan_workspace_bytes(const thff_state_shape* shape) {
    return guarded([&]() -> long long {
        StateShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? state_workspace_bytes(s) : rc;
    });
}

THFF_TWINS(thff_state_scan,
           (const thff_state_shape* shape, const void* d_x, const void* d_delta, const void* d_a, const void* d_b,
            const void* d_c, const void* d_skip, const void* d_gate, const void* d_delta_bias, void* d_y,
            const void* d_state_in, void* d_state_out, const void* d_slots, const void* d_lengths, void* d_saved,
            void* d_workspace, void* stream),
           state_impl(shape,
                      StateForward{d_x, d_delta, floats(d_a), d_b, d_c, floats(d_skip), d_gate, floats(d_delta_bias),
                                   floats(d_state_in), ints(d_slots), ints(d_lengths), d_y, floats(d_state_out),
                                   floats(d_saved), floats(d_workspace)},
                      stream, synchronize))

THFF_TWINS(thff_state_scan_backward,
           (const thff_state_shape* shape, const thff_state_gradients* arrays, void* d_workspace, void* stream),
           state_backward_impl(shape, arrays, d_workspace, stream, synchronize))

THFF_TWINS(thff_rms_norm,
           (int precision, const void* d_x, long long x_stride, const void* d_residual, long long residual_stride,
            const void* d_weight, float eps, void* d_y, long long y_stride, void* d_sum, long long sum_stride,
            void* d_rstd, long long rows, int cols, void* stream),
           rms_impl(RmsForward{precision, rows, cols, d_x, x_stride, d_residual, residual_stride, floats(d_weight), eps,
                               d_y, y_stride, nullptr, 0, d_sum, sum_stride, floats(d_rstd)},
                    stream, synchronize))

THFF_TWINS(thff_rms_norm_8bit,
           (int precision, const void* d_x, long long x_stride, const void* d_residual, long long residual_stride,
            const void* d_weight, float eps, void* d_q, long long q_stride, void* d_scales, int block, void* d_sum,
            long long sum_stride, long long rows, int cols, void* stream),
           rms_8bit(RmsForward{precision, rows, cols, d_x, x_stride, d_residual, residual_stride, floats(d_weight), eps,
                               d_q, q_stride, floats(d_scales), block, d_sum, sum_stride, nullptr},
                    stream, synchronize))

long long thff_rms_norm_workspace_bytes(long long rows, int cols) {
    return guarded([&]() -> long long {
        const int rc = check_rms(THFF_FLOAT, rows, cols);
        return rc == THFF_OK ? rms_workspace_bytes(rows, cols) : rc;
    });
}

THFF_TWINS(thff_rms_norm_backward,
           (int precision, const void* d_dy, long long dy_stride, const void* d_sum, long long sum_stride,
            const void* d_rstd, const void* d_weight, const void* d_dsum, long long dsum_stride, void* d_dx,
            long long dx_stride, void* d_dweight, void* d_workspace, long long rows, int cols, void* stream),
           rms_backward_impl(RmsBackward{precision, rows, cols, d_dy, dy_stride, d_sum, sum_stride, floats(d_rstd),
                                         floats(d_weight), d_dsum, dsum_stride, d_dx, dx_stride, floats(d_dweight),
                                         floats(d_workspace)},
                             stream, synchronize))

}  // extern "C"
