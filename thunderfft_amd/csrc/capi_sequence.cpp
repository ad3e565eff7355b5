// capi_sequence.cpp -- the C ABI of the sequence operators of
// include/thunderfft/thunderfft.h: argument checks, all before any HIP call, and dispatch.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "errors.hpp"
#include "sequence.hpp"
#include "thunderfft/thunderfft.h"

namespace {

using thff::fail;
using thff::fail_hip;
using thff::ScanShape;

constexpr int kMostSize = 1 << 30;
// Elements of a strided buffer: byte offsets stay within 63 bits.
constexpr __int128 kMostSpan = static_cast<__int128>(1) << 60;

bool value_type(int p) { return p == THFF_FLOAT || p == THFF_HALF || p == THFF_BFLOAT16; }

bool aligned(const void* p, unsigned bytes) {
    return reinterpret_cast<std::uintptr_t>(p) % bytes == 0;
}

// Fills a stride of 0 in; false: rows of `length` would overlap, or the offsets overflow.
bool stride_of(long long given, long long length, long long rows, long long* stride) {
    *stride = given ? given : length;
    return *stride >= length && static_cast<__int128>(rows) * *stride <= kMostSpan;
}

int check_shape(const thff_scan_shape* shape, ScanShape* out) {
    if (!shape) return fail(THFF_EINVAL, "thff_scan_shape is null");
    if (!value_type(shape->precision))
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan supports float, half and bfloat16 only");
    if (shape->layout != THFF_CHANNELS_LAST && shape->layout != THFF_CHANNELS_FIRST)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan layout must be channels last or first");
    if (shape->batch < 0 || shape->n < 0 || shape->channels < 0)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan batch, n and channels must be nonnegative");
    if (shape->batch > kMostSize || shape->n > kMostSize || shape->channels > kMostSize)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan batch, n and channels must be at most 2^30");
    const bool first = shape->layout == THFF_CHANNELS_FIRST;
    *out = ScanShape{shape->precision, first, shape->batch, shape->n, shape->channels,
                     shape->states, 0, 0, 0};
    const long long length = first ? shape->n : shape->channels;
    const long long rows =
        static_cast<long long>(shape->batch) * (first ? shape->channels : shape->n);
    if (!stride_of(shape->x_stride, length, rows, &out->x_stride) ||
        !stride_of(shape->gate_stride, length, rows, &out->gate_stride) ||
        !stride_of(shape->y_stride, length, rows, &out->y_stride))
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan stride is shorter than a row or too long");
    if (!thff::scan_fits(*out))
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan shape exceeds one launch");
    return THFF_OK;
}

unsigned element_bytes(int precision) { return precision == THFF_FLOAT ? 4 : 2; }

int finish(hipError_t err, hipStream_t s, bool synchronize, const char* who) {
    if (err != hipSuccess) return fail_hip(err, who);
    if (!synchronize) return THFF_OK;
    err = hipStreamSynchronize(s);
    return err == hipSuccess ? THFF_OK : fail_hip(err, who);
}

int scan_impl(const thff_scan_shape* shape, const void* x, const void* gate, void* y,
              const void* state_in, void* state_out, const void* slots, const void* lengths,
              void* saved, void* workspace, void* stream, bool synchronize) {
    ScanShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (s.batch == 0 || s.channels == 0) return THFF_OK;
    if (s.n > 0) {
        if (!x || !gate || !y)
            return fail(THFF_EINVAL, "ThunderFFT_gated_scan requires non-null x, gate and y");
        if (y == x || y == gate)
            return fail(THFF_EINVAL, "ThunderFFT_gated_scan output must not alias its inputs");
        const unsigned e = element_bytes(s.precision);
        if (!aligned(x, e) || !aligned(gate, e) || !aligned(y, e))
            return fail(THFF_EINVAL, "ThunderFFT_gated_scan requires element-aligned buffers");
    }
    if (!aligned(state_in, 4) || !aligned(state_out, 4) || !aligned(slots, 4) ||
        !aligned(lengths, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_gated_scan requires 4-byte aligned states, slots and lengths");
    if (slots && s.states < 0)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan states must be nonnegative");
    if (!aligned(saved, 16) || !aligned(workspace, 16))
        return fail(THFF_EINVAL,
                    "ThunderFFT_gated_scan requires 16-byte aligned saved and workspace");
    if (!workspace && thff::scan_workspace_bytes(s) > 0)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan requires a workspace of " +
                                     std::to_string(thff::scan_workspace_bytes(s)) + " bytes");
    const thff::ScanForward a{x,
                              gate,
                              static_cast<const float*>(state_in),
                              static_cast<const int*>(slots),
                              static_cast<const int*>(lengths),
                              y,
                              static_cast<float*>(state_out),
                              static_cast<float*>(saved),
                              workspace};
    auto st = static_cast<hipStream_t>(stream);
    return finish(thff::launch_gated_scan(s, a, st), st, synchronize, "ThunderFFT_gated_scan");
}

int scan_backward_impl(const thff_scan_shape* shape, const void* dy, const void* x,
                       const void* gate, const void* saved, const void* dstate_out,
                       const void* lengths, void* dx, void* dgate, void* dstate_in,
                       void* workspace, void* stream, bool synchronize) {
    ScanShape s;
    const int rc = check_shape(shape, &s);
    if (rc != THFF_OK) return rc;
    if (s.batch == 0 || s.channels == 0) return THFF_OK;
    if (s.n > 0) {
        if (!dy || !x || !gate || !dx || !dgate)
            return fail(THFF_EINVAL,
                        "ThunderFFT_gated_scan_backward requires non-null dy, x, gate, dx and dgate");
        if (dx == dgate || dx == dy || dx == x || dx == gate || dgate == dy || dgate == x ||
            dgate == gate)
            return fail(THFF_EINVAL,
                        "ThunderFFT_gated_scan_backward outputs must not alias its inputs");
        const unsigned e = element_bytes(s.precision);
        if (!aligned(dy, e) || !aligned(x, e) || !aligned(gate, e) || !aligned(dx, e) ||
            !aligned(dgate, e))
            return fail(THFF_EINVAL,
                        "ThunderFFT_gated_scan_backward requires element-aligned buffers");
        if (!saved && thff::scan_saved_bytes(s) > 0)
            return fail(THFF_EINVAL,
                        "ThunderFFT_gated_scan_backward requires what the forward call saved");
    }
    if (!aligned(dstate_out, 4) || !aligned(dstate_in, 4) || !aligned(lengths, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_gated_scan_backward requires 4-byte aligned states and lengths");
    if (!aligned(saved, 16) || !aligned(workspace, 16))
        return fail(THFF_EINVAL,
                    "ThunderFFT_gated_scan_backward requires 16-byte aligned saved and workspace");
    if (!workspace && thff::scan_workspace_bytes(s) > 0)
        return fail(THFF_EINVAL, "ThunderFFT_gated_scan_backward requires a workspace of " +
                                     std::to_string(thff::scan_workspace_bytes(s)) + " bytes");
    const thff::ScanBackward a{dy,
                               x,
                               gate,
                               static_cast<const float*>(saved),
                               static_cast<const float*>(dstate_out),
                               static_cast<const int*>(lengths),
                               dx,
                               dgate,
                               static_cast<float*>(dstate_in),
                               workspace};
    auto st = static_cast<hipStream_t>(stream);
    return finish(thff::launch_gated_scan_backward(s, a, st), st, synchronize,
                  "ThunderFFT_gated_scan_backward");
}

int check_norm(int precision, long long rows, int cols) {
    if (!value_type(precision))
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm supports float, half and bfloat16 only");
    if (rows < 0) return fail(THFF_EINVAL, "ThunderFFT_layer_norm rows must be nonnegative");
    if (cols < 1 || cols > kMostSize)
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm cols must be 1 to 2^30");
    return THFF_OK;
}

int norm_impl(int precision, const void* x, long long x_stride, const void* weight,
              const void* bias, float eps, void* y, long long y_stride, void* mean, void* rstd,
              long long rows, int cols, void* stream, bool synchronize) {
    const int rc = check_norm(precision, rows, cols);
    if (rc != THFF_OK) return rc;
    if (!(eps >= 0.0f)) return fail(THFF_EINVAL, "ThunderFFT_layer_norm eps must be nonnegative");
    thff::NormForward a{precision, rows, cols, x, 0, static_cast<const float*>(weight),
                        static_cast<const float*>(bias), eps, y, 0, static_cast<float*>(mean),
                        static_cast<float*>(rstd)};
    if (!stride_of(x_stride, cols, rows, &a.x_stride) ||
        !stride_of(y_stride, cols, rows, &a.y_stride))
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm stride is shorter than a row or too long");
    if (rows == 0) return THFF_OK;
    if (!x || !y) return fail(THFF_EINVAL, "ThunderFFT_layer_norm requires non-null x and y");
    if (y == x) return fail(THFF_EINVAL, "ThunderFFT_layer_norm output must not alias its input");
    const unsigned e = element_bytes(precision);
    if (!aligned(x, e) || !aligned(y, e))
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm requires element-aligned buffers");
    if (!aligned(weight, 4) || !aligned(bias, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_layer_norm requires 4-byte aligned weights and statistics");
    auto st = static_cast<hipStream_t>(stream);
    return finish(thff::launch_layer_norm(a, st), st, synchronize, "ThunderFFT_layer_norm");
}

int norm_backward_impl(int precision, const void* dy, long long dy_stride, const void* x,
                       long long x_stride, const void* mean, const void* rstd, const void* weight,
                       void* dx, long long dx_stride, void* dweight, void* dbias, void* workspace,
                       long long rows, int cols, void* stream, bool synchronize) {
    const int rc = check_norm(precision, rows, cols);
    if (rc != THFF_OK) return rc;
    thff::NormBackward a{precision,
                         rows,
                         cols,
                         dy,
                         0,
                         x,
                         0,
                         static_cast<const float*>(mean),
                         static_cast<const float*>(rstd),
                         static_cast<const float*>(weight),
                         dx,
                         0,
                         static_cast<float*>(dweight),
                         static_cast<float*>(dbias),
                         static_cast<float*>(workspace)};
    if (!stride_of(dy_stride, cols, rows, &a.dy_stride) ||
        !stride_of(x_stride, cols, rows, &a.x_stride) ||
        !stride_of(dx_stride, cols, rows, &a.dx_stride))
        return fail(THFF_EINVAL,
                    "ThunderFFT_layer_norm_backward stride is shorter than a row or too long");
    if (rows == 0 && !dweight && !dbias) return THFF_OK;
    if (rows > 0) {
        if (!dy || !x || !mean || !rstd || !dx)
            return fail(THFF_EINVAL,
                        "ThunderFFT_layer_norm_backward requires non-null dy, x, mean, rstd and dx");
        if (dx == dy || dx == x)
            return fail(THFF_EINVAL,
                        "ThunderFFT_layer_norm_backward output must not alias its inputs");
        const unsigned e = element_bytes(precision);
        if (!aligned(dy, e) || !aligned(x, e) || !aligned(dx, e))
            return fail(THFF_EINVAL,
                        "ThunderFFT_layer_norm_backward requires element-aligned buffers");
        if (!workspace && (dweight || dbias) && thff::norm_workspace_bytes(rows, cols) > 0)
            return fail(THFF_EINVAL,
                        "ThunderFFT_layer_norm_backward requires a workspace of " +
                            std::to_string(thff::norm_workspace_bytes(rows, cols)) + " bytes");
    }
    if (dweight && dweight == dbias)
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm_backward dweight must not alias dbias");
    if (!aligned(weight, 4) || !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(dweight, 4) ||
        !aligned(dbias, 4))
        return fail(THFF_EINVAL,
                    "ThunderFFT_layer_norm_backward requires 4-byte aligned weights and statistics");
    if (!aligned(workspace, 16))
        return fail(THFF_EINVAL, "ThunderFFT_layer_norm_backward requires a 16-byte aligned workspace");
    auto st = static_cast<hipStream_t>(stream);
    return finish(thff::launch_layer_norm_backward(a, st), st, synchronize,
                  "ThunderFFT_layer_norm_backward");
}

// Nothing is thrown through the C ABI (a message's allocation may fail).
template <class F>
auto guarded(F f) noexcept -> decltype(f()) {
    try {
        return f();
    } catch (...) {
        return THFF_EIO;
    }
}

}  // namespace

extern "C" {

long long thff_gated_scan_saved_bytes(const thff_scan_shape* shape) {
    return guarded([&]() -> long long {
        ScanShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? thff::scan_saved_bytes(s) : rc;
    });
}

long long thff_gated_scan_workspace_bytes(const thff_scan_shape* shape) {
    return guarded([&]() -> long long {
        ScanShape s;
        const int rc = check_shape(shape, &s);
        return rc == THFF_OK ? thff::scan_workspace_bytes(s) : rc;
    });
}

int thff_gated_scan(const thff_scan_shape* shape, const void* d_x, const void* d_gate, void* d_y,
                    const void* d_state_in, void* d_state_out, const void* d_slots,
                    const void* d_lengths, void* d_saved, void* d_workspace, void* stream) {
    return guarded([&] {
        return scan_impl(shape, d_x, d_gate, d_y, d_state_in, d_state_out, d_slots, d_lengths, d_saved,
                         d_workspace, stream, true);
    });
}

int thff_gated_scan_async(const thff_scan_shape* shape, const void* d_x, const void* d_gate,
                          void* d_y, const void* d_state_in, void* d_state_out,
                          const void* d_slots, const void* d_lengths, void* d_saved,
                          void* d_workspace, void* stream) {
    return guarded([&] {
        return scan_impl(shape, d_x, d_gate, d_y, d_state_in, d_state_out, d_slots, d_lengths, d_saved,
                         d_workspace, stream, false);
    });
}

int thff_gated_scan_backward(const thff_scan_shape* shape, const void* d_dy, const void* d_x,
                             const void* d_gate, const void* d_saved, const void* d_dstate_out,
                             const void* d_lengths, void* d_dx, void* d_dgate, void* d_dstate_in,
                             void* d_workspace, void* stream) {
    return guarded([&] {
        return scan_backward_impl(shape, d_dy, d_x, d_gate, d_saved, d_dstate_out, d_lengths, d_dx,
                                  d_dgate, d_dstate_in, d_workspace, stream, true);
    });
}

int thff_gated_scan_backward_async(const thff_scan_shape* shape, const void* d_dy,
                                   const void* d_x, const void* d_gate, const void* d_saved,
                                   const void* d_dstate_out, const void* d_lengths, void* d_dx,
                                   void* d_dgate, void* d_dstate_in, void* d_workspace,
                                   void* stream) {
    return guarded([&] {
        return scan_backward_impl(shape, d_dy, d_x, d_gate, d_saved, d_dstate_out, d_lengths, d_dx,
                                  d_dgate, d_dstate_in, d_workspace, stream, false);
    });
}

int thff_layer_norm(int precision, const void* d_x, long long x_stride, const void* d_weight,
                    const void* d_bias, float eps, void* d_y, long long y_stride, void* d_mean,
                    void* d_rstd, long long rows, int cols, void* stream) {
    return guarded([&] {
        return norm_impl(precision, d_x, x_stride, d_weight, d_bias, eps, d_y, y_stride, d_mean, d_rstd,
                         rows, cols, stream, true);
    });
}

int thff_layer_norm_async(int precision, const void* d_x, long long x_stride,
                          const void* d_weight, const void* d_bias, float eps, void* d_y,
                          long long y_stride, void* d_mean, void* d_rstd, long long rows, int cols,
                          void* stream) {
    return guarded([&] {
        return norm_impl(precision, d_x, x_stride, d_weight, d_bias, eps, d_y, y_stride, d_mean, d_rstd,
                         rows, cols, stream, false);
    });
}

long long thff_layer_norm_workspace_bytes(long long rows, int cols) {
    return guarded([&]() -> long long {
        const int rc = check_norm(THFF_FLOAT, rows, cols);
        return rc == THFF_OK ? thff::norm_workspace_bytes(rows, cols) : rc;
    });
}

int thff_layer_norm_backward(int precision, const void* d_dy, long long dy_stride,
                             const void* d_x, long long x_stride, const void* d_mean,
                             const void* d_rstd, const void* d_weight, void* d_dx,
                             long long dx_stride, void* d_dweight, void* d_dbias,
                             void* d_workspace, long long rows, int cols, void* stream) {
    return guarded([&] {
        return norm_backward_impl(precision, d_dy, dy_stride, d_x, x_stride, d_mean, d_rstd, d_weight,
                                  d_dx, dx_stride, d_dweight, d_dbias, d_workspace, rows, cols, stream,
                                  true);
    });
}

int thff_layer_norm_backward_async(int precision, const void* d_dy, long long dy_stride,
                                   const void* d_x, long long x_stride, const void* d_mean,
                                   const void* d_rstd, const void* d_weight, void* d_dx,
                                   long long dx_stride, void* d_dweight, void* d_dbias,
                                   void* d_workspace, long long rows, int cols, void* stream) {
    return guarded([&] {
        return norm_backward_impl(precision, d_dy, dy_stride, d_x, x_stride, d_mean, d_rstd, d_weight,
                                  d_dx, dx_stride, d_dweight, d_dbias, d_workspace, rows, cols, stream,
                                  false);
    });
}

}  // extern "C"
