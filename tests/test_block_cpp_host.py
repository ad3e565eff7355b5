"""The C++ templates of a state space block's operators: instantiated for every type by a host compiler
and by hipcc, and their arguments handed on in the C ABI's order.  No GPU: every refusal comes before
any HIP call."""
import os
import subprocess

import pytest

from test_sequence_cpp_host import PROGRAM as SEQUENCE
from test_sequence_cpp_host import ROCM, ROOT, TYPES, hipcc

# Each call has one wrong argument, whose message tells it from the others.
PROGRAM = SEQUENCE[:SEQUENCE.index("template <class T, class Other>")] + r"""
template <class T, class Other>
void conv() {
    const auto s = ThunderFFT_conv_shape<T>(2, 300, 70, 4);
    if (s.batch != 2 || s.n != 300 || s.channels != 70 || s.width != 4 || s.states != 2 || s.silu != 1 || s.x_stride || s.y_stride)
        std::printf("conv shape\n");
    if (ThunderFFT_conv_shape<T>(2, 300, 70, 4, false).silu != 0) std::printf("silu\n");
    if (!ThunderFFT_short_conv_workspace_bytes(s)) std::printf("conv workspace bytes\n");
    auto bad = s;
    bad.n = -1;
    refused("nonnegative", [&] { ThunderFFT_short_conv_workspace_bytes(bad); });
    T *x = at<T>(1), *y = at<T>(2), *first = at<T>(3), *last = at<T>(4);
    float *w = at<float>(5), *b = at<float>(6);
    int *slots = at<int>(7), *lengths = at<int>(8);
    char* work = at<char>(9);
    refused("another type", [&] { ThunderFFT_short_conv<T>(ThunderFFT_conv_shape<Other>(2, 300, 70, 4), x, w, b, y, first, last, slots, lengths); });
    refused("non-null", [&] { ThunderFFT_short_conv<T>(s, nullptr, w, b, y, first, last, slots, lengths); });
    refused("non-null", [&] { ThunderFFT_short_conv<T>(s, x, nullptr, b, y, first, last, slots, lengths); });
    refused("alias", [&] { ThunderFFT_short_conv<T>(s, x, w, b, x, first, last, slots, lengths); });
    refused("alias", [&] { ThunderFFT_short_conv<T>(s, x, w, b, first, first, last, slots, lengths); });
    refused("alias", [&] { ThunderFFT_short_conv<T>(s, x, w, b, last, first, last, slots, lengths); });
    refused("element-aligned", [&] { ThunderFFT_short_conv<T>(s, x, w, b, y, off(first, 1), last, slots, lengths); });
    refused("element-aligned", [&] { ThunderFFT_short_conv<T>(s, x, w, b, y, first, off(last, 1), slots, lengths); });
    refused("4-byte", [&] { ThunderFFT_short_conv<T>(s, x, w, off(b, 2), y, first, last, slots, lengths); });
    refused("4-byte", [&] { ThunderFFT_short_conv<T>(s, x, w, b, y, first, last, off(slots, 2), lengths); });
    refused("4-byte", [&] { ThunderFFT_short_conv<T>(s, x, w, b, y, first, last, slots, off(lengths, 2)); });

    T *dy = at<T>(10), *dx = at<T>(11), *dlast = at<T>(12), *dfirst = at<T>(13);
    float *dw = at<float>(14), *db = at<float>(15);
    const auto back = [&](T* dy, T* x, float* w, float* b, T* first, T* dlast, int* lengths, T* dx, float* dw, float* db, T* dfirst,
                          void* work) {
        ThunderFFT_short_conv_backward<T>(s, dy, x, w, b, first, dlast, lengths, dx, dw, db, dfirst, work);
    };
    refused("another type", [&] { ThunderFFT_short_conv_backward<T>(ThunderFFT_conv_shape<Other>(2, 300, 70, 4), dy, x, w, b, first, dlast, lengths, dx, dw, db, dfirst, work); });
    refused("non-null", [&] { back(nullptr, x, w, b, first, dlast, lengths, dx, dw, db, dfirst, work); });
    refused("alias", [&] { back(dy, x, w, b, first, dlast, lengths, dy, dw, db, dfirst, work); });
    refused("alias", [&] { back(dy, x, w, b, first, dlast, lengths, dx, dw, db, first, work); });
    refused("alias", [&] { back(dy, x, w, b, first, dlast, lengths, dx, dw, db, dlast, work); });
    refused("alias", [&] { back(dy, x, w, b, first, dlast, lengths, dx, w, db, dfirst, work); });
    refused("alias", [&] { back(dy, x, w, b, first, dlast, lengths, dx, dw, b, dfirst, work); });
    refused("4-byte", [&] { back(dy, x, w, b, first, dlast, off(lengths, 2), dx, dw, db, dfirst, work); });
    refused("requires a workspace", [&] { back(dy, x, w, b, first, dlast, lengths, dx, dw, db, dfirst, nullptr); });
    refused("16-byte", [&] { back(dy, x, w, b, first, dlast, lengths, dx, dw, db, dfirst, work + 4); });
}

template <class T, class Other>
void state() {
    const auto s = ThunderFFT_state_shape<T>(2, 300, 70, 16, 2);
    if (s.batch != 2 || s.n != 300 || s.channels != 70 || s.order != 16 || s.groups != 2 || s.states != 2 || s.x_stride ||
        s.delta_stride || s.gate_stride || s.b_stride || s.c_stride || s.y_stride)
        std::printf("state shape\n");
    // A state of 16 values a channel for every 16 steps.
    if (ThunderFFT_state_scan_saved_bytes(s) != 4 * 2 * 19 * 70 * 16) std::printf("saved bytes\n");
    if (!ThunderFFT_state_scan_forward_bytes(s) || ThunderFFT_state_scan_workspace_bytes(s) < ThunderFFT_state_scan_forward_bytes(s))
        std::printf("state workspace bytes\n");
    auto bad = s;
    bad.order = 65;
    refused("order", [&] { ThunderFFT_state_scan_saved_bytes(bad); });
    refused("order", [&] { ThunderFFT_state_scan_forward_bytes(bad); });
    refused("order", [&] { ThunderFFT_state_scan_workspace_bytes(bad); });
    T *x = at<T>(1), *delta = at<T>(2), *b = at<T>(3), *c = at<T>(4), *gate = at<T>(5), *y = at<T>(6);
    float *a = at<float>(7), *skip = at<float>(8), *bias = at<float>(9), *first = at<float>(10), *last = at<float>(11);
    int *slots = at<int>(12), *lengths = at<int>(13);
    char *saved = at<char>(14), *work = at<char>(15);
    const auto call = [&](const thff_state_shape& s, T* x, T* delta, float* a, T* b, T* c, float* skip, T* gate, float* bias, T* y,
                          float* first, float* last, int* slots, int* lengths, void* saved, void* work) {
        ThunderFFT_state_scan<T>(s, x, delta, a, b, c, skip, gate, bias, y, first, last, slots, lengths, saved, work);
    };
    refused("another type", [&] { call(ThunderFFT_state_shape<Other>(2, 300, 70, 16, 2), x, delta, a, b, c, skip, gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("non-null", [&] { call(s, x, delta, nullptr, b, c, skip, gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("non-null", [&] { call(s, x, delta, a, b, nullptr, skip, gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("element-aligned", [&] { call(s, x, off(delta, 1), a, b, c, skip, gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("element-aligned", [&] { call(s, x, delta, a, off(b, 1), c, skip, gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("element-aligned", [&] { call(s, x, delta, a, b, c, skip, off(gate, 1), bias, y, first, last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, off(skip, 2), gate, bias, y, first, last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, skip, gate, off(bias, 2), y, first, last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, off(first, 2), last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, first, off(last, 2), slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, first, last, off(slots, 2), lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, first, last, slots, off(lengths, 2), saved, work); });
    refused("alias", [&] { call(s, x, delta, a, b, c, skip, gate, bias, gate, first, last, slots, lengths, saved, work); });
    refused("16-byte", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, first, last, slots, lengths, saved + 4, work); });
    refused("requires a workspace", [&] { call(s, x, delta, a, b, c, skip, gate, bias, y, first, last, slots, lengths, saved, nullptr); });

    using G = ThunderFFT_state_gradients<T>;
    const G good{at<T>(16), x, delta, a, b, c, skip, gate, bias, saved, first, lengths, at<T>(17), at<T>(18), at<float>(19),
                 at<T>(20), at<T>(21), at<float>(22), at<T>(23), at<float>(24), at<float>(25)};
    const auto with = [&](const char* what, auto change) {
        G g = good;
        change(g);
        refused(what, [&] { ThunderFFT_state_scan_backward<T>(s, g, work); });
    };
    refused("another type", [&] { ThunderFFT_state_scan_backward<T>(ThunderFFT_state_shape<Other>(2, 300, 70, 16, 2), good, work); });
    refused("requires a workspace", [&] { ThunderFFT_state_scan_backward<T>(s, good, nullptr); });
    with("non-null da", [](G& g) { g.da = nullptr; });
    with("non-null dy", [](G& g) { g.dy = nullptr; });
    with("requires dgate", [](G& g) { g.dgate = nullptr; });
    with("forward call saved", [](G& g) { g.saved = nullptr; });
    with("alias", [](G& g) { g.dx = const_cast<T*>(g.dy); });
    with("alias", [](G& g) { g.ddelta = const_cast<T*>(g.delta); });
    with("alias", [](G& g) { g.da = const_cast<float*>(g.a); });
    with("alias", [](G& g) { g.db = const_cast<T*>(g.c); });
    with("alias", [](G& g) { g.dc = g.db; });
    with("alias", [](G& g) { g.dskip = const_cast<float*>(g.skip); });
    with("alias", [](G& g) { g.dgate = const_cast<T*>(g.gate); });
    with("alias", [](G& g) { g.ddelta_bias = const_cast<float*>(g.delta_bias); });
    with("alias", [](G& g) { g.dstate_in = const_cast<float*>(g.dstate_out); });
    with("4-byte", [](G& g) { g.lengths = off(g.lengths, 2); });
    with("4-byte", [](G& g) { g.skip = off(g.skip, 2); });
    with("element-aligned", [](G& g) { g.x = off(g.x, 1); });
    with("16-byte", [](G& g) { g.saved = static_cast<const char*>(g.saved) + 4; });
}

template <class T>
void rms() {
    T *x = at<T>(1), *r = at<T>(2), *y = at<T>(3), *sum = at<T>(4), *dy = at<T>(5), *dx = at<T>(6), *dsum = at<T>(7);
    float *w = at<float>(8), *rstd = at<float>(9), *scales = at<float>(10), *dw = at<float>(11);
    unsigned char* q = at<unsigned char>(12);
    char* work = at<char>(13);
    refused("non-null", [&] { ThunderFFT_rms_norm<T>(nullptr, r, w, 1e-5f, y, sum, 4, 8, rstd); });
    refused("alias", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, x, sum, 4, 8, rstd); });
    refused("alias", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, r, sum, 4, 8, rstd); });
    refused("alias", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, x, 4, 8, rstd); });
    refused("eps", [&] { ThunderFFT_rms_norm<T>(x, r, w, -1.0f, y, sum, 4, 8, rstd); });
    refused("rows", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, -4, 8, rstd); });
    refused("cols", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 0, rstd); });
    refused("4-byte", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 8, off(rstd, 2)); });
    refused("stride", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 8, rstd, 7); });
    refused("stride", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 8, rstd, 8, 7); });
    refused("stride", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 8, rstd, 8, 8, 7); });
    refused("stride", [&] { ThunderFFT_rms_norm<T>(x, r, w, 1e-5f, y, sum, 4, 8, rstd, 8, 8, 8, 7); });
    refused("block must be", [&] { ThunderFFT_rms_norm_8bit<T>(x, r, w, 1e-5f, q, scales, 64, sum, 4, 256); });
    refused("scales", [&] { ThunderFFT_rms_norm_8bit<T>(x, r, w, 1e-5f, q, nullptr, 128, sum, 4, 256); });
    refused("non-null", [&] { ThunderFFT_rms_norm_8bit<T>(x, r, w, 1e-5f, nullptr, scales, 128, sum, 4, 256); });
    refused("rows", [&] { ThunderFFT_rms_norm_8bit<T>(x, r, w, 1e-5f, q, scales, 128, sum, -4, 256); });
    refused("stride", [&] { ThunderFFT_rms_norm_8bit<T>(x, r, w, 1e-5f, q, scales, 128, sum, 4, 256, 0, 0, 255); });
    if (ThunderFFT_rms_norm_workspace_bytes(300, 64) != 4 * 256 * 64) std::printf("rms workspace bytes\n");
    const auto back = [&](T* dy, T* sum, float* rstd, float* w, T* dsum, T* dx, float* dw, void* work, long long a = 0, long long b = 0,
                          long long c = 0, long long d = 0) {
        ThunderFFT_rms_norm_backward<T>(dy, sum, rstd, w, dsum, dx, dw, work, 4, 8, a, b, c, d);
    };
    refused("non-null", [&] { back(dy, sum, nullptr, w, dsum, dx, dw, work); });
    refused("alias", [&] { back(dy, sum, rstd, w, dsum, dy, dw, work); });
    refused("alias", [&] { back(dy, sum, rstd, w, dsum, dsum, dw, work); });
    refused("alias", [&] { back(dy, sum, rstd, w, dsum, dx, w, work); });
    refused("4-byte", [&] { back(dy, sum, rstd, off(w, 2), dsum, dx, dw, work); });
    refused("element-aligned", [&] { back(dy, sum, rstd, w, off(dsum, 1), dx, dw, work); });
    refused("requires a workspace", [&] { back(dy, sum, rstd, w, dsum, dx, dw, nullptr); });
    refused("stride", [&] { back(dy, sum, rstd, w, dsum, dx, dw, work, 7); });
    refused("stride", [&] { back(dy, sum, rstd, w, dsum, dx, dw, work, 8, 7); });
    refused("stride", [&] { back(dy, sum, rstd, w, dsum, dx, dw, work, 8, 8, 7); });
    refused("stride", [&] { back(dy, sum, rstd, w, dsum, dx, dw, work, 8, 8, 8, 7); });
}

int main() {
    conv<float, half>();
    conv<half, __hip_bfloat16>();
    conv<__hip_bfloat16, float>();
    state<float, half>();
    state<half, __hip_bfloat16>();
    state<__hip_bfloat16, float>();
    rms<float>();
    rms<half>();
    rms<__hip_bfloat16>();
    std::puts("done");
}
"""


def test_templates_hand_their_arguments_on(tmp_path):
    import thunderfft_amd as thff

    thff.lib()
    src, exe = tmp_path / "calls.cpp", tmp_path / "calls"
    src.write_text(PROGRAM)
    folder = os.path.dirname(thff.LIB_PATH)
    res = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"),
                          "-isystem", os.path.join(ROCM, "include"), str(src), "-o", str(exe), "-L", folder,
                          "-lthunderfft_amd", f"-Wl,-rpath,{folder}", "-L", os.path.join(ROCM, "lib"), "-lamdhip64",
                          f"-Wl,-rpath,{os.path.join(ROCM, 'lib')}"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "done\n", (res.stdout, res.stderr)


def test_templates_compile_for_the_gpu(tmp_path):
    body = "".join(f"""
template void thunderfft::ThunderFFT_short_conv<{T}>(const thff_conv_shape&, const {T}*, const float*, const float*, {T}*,
    const {T}*, {T}*, const int*, const int*, hipStream_t);
template void thunderfft::ThunderFFT_state_scan_backward<{T}>(const thff_state_shape&,
    const thunderfft::ThunderFFT_state_gradients<{T}>&, void*, hipStream_t);
template void thunderfft::ThunderFFT_rms_norm_8bit<{T}>(const {T}*, const {T}*, const float*, float, unsigned char*, float*, int,
    {T}*, long long, int, long long, long long, long long, long long, hipStream_t);
""" for T in TYPES)
    src = tmp_path / "k.hip"
    src.write_text(f"#include <hip/hip_bf16.h>\n#include <thunderfft/thunderfft.hpp>\n{body}")
    command = [hipcc(), "--offload-arch=gfx950", "-std=c++17", "-fsyntax-only", "-I", os.path.join(ROOT, "include")]
    res = subprocess.run([*command, str(src)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
