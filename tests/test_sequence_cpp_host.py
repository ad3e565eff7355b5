"""The C++ templates of the sequence operators: instantiated for every type by a host compiler and
by hipcc, and their arguments handed on in the C ABI's order.  No GPU: every refusal comes before
any HIP call."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
TYPES = ("float", "half", "__hip_bfloat16")

# Each call has one wrong argument, whose message tells it from the others.
PROGRAM = r"""
#include <thunderfft/thunderfft.hpp>

#include <cstdio>
#include <cstring>

using namespace thunderfft;

template <class F>
void refused(const char* what, F call) {
    try {
        call();
        std::printf("not refused: %s\n", what);
    } catch (const std::invalid_argument& e) {
        if (!std::strstr(e.what(), what)) std::printf("\"%s\" is not \"%s\"\n", e.what(), what);
    }
}

template <class T>
T* at(unsigned long long v) {
    return reinterpret_cast<T*>(v << 16);  // never dereferenced
}

template <class P>
P* off(P* p, int bytes) {
    return reinterpret_cast<P*>(reinterpret_cast<char*>(const_cast<std::remove_const_t<P>*>(p)) + bytes);
}

template <class T, class Other>
void scan() {
    const auto s = ThunderFFT_scan_shape<T>(2, 300, 70);
    if (s.batch != 2 || s.n != 300 || s.channels != 70 || s.states != 2 || s.layout != THFF_CHANNELS_LAST ||
        s.x_stride || s.gate_stride || s.y_stride)
        std::printf("shape\n");
    if (ThunderFFT_scan_shape<T>(2, 300, 70, true).layout != THFF_CHANNELS_FIRST) std::printf("layout\n");
    // 300 steps: a state for every 56 of them.
    if (ThunderFFT_gated_scan_saved_bytes(s) != 4 * 2 * 70 * 6) std::printf("saved bytes\n");
    if (!ThunderFFT_gated_scan_workspace_bytes(s)) std::printf("workspace bytes\n");
    auto bad = s;
    bad.n = -1;
    refused("nonnegative", [&] { ThunderFFT_gated_scan_saved_bytes(bad); });
    refused("nonnegative", [&] { ThunderFFT_gated_scan_workspace_bytes(bad); });

    T *x = at<T>(1), *gate = at<T>(2), *y = at<T>(3);
    float *first = at<float>(4), *last = at<float>(5);
    int *slots = at<int>(6), *lengths = at<int>(7);
    char *saved = at<char>(8), *work = at<char>(9);
    const auto call = [&](const thff_scan_shape& shape, T* x, T* gate, T* y, float* first, float* last, int* slots,
                          int* lengths, void* saved, void* work) {
        ThunderFFT_gated_scan<T>(shape, x, gate, y, first, last, slots, lengths, saved, work);
    };
    refused("another type", [&] { call(ThunderFFT_scan_shape<Other>(2, 300, 70), x, gate, y, first, last, slots, lengths, saved, work); });
    refused("non-null", [&] { call(s, nullptr, gate, y, first, last, slots, lengths, saved, work); });
    refused("non-null", [&] { call(s, x, nullptr, y, first, last, slots, lengths, saved, work); });
    refused("non-null", [&] { call(s, x, gate, nullptr, first, last, slots, lengths, saved, work); });
    refused("alias", [&] { call(s, x, gate, x, first, last, slots, lengths, saved, work); });
    refused("alias", [&] { call(s, x, gate, gate, first, last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, gate, y, off(first, 2), last, slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, gate, y, first, off(last, 2), slots, lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, gate, y, first, last, off(slots, 2), lengths, saved, work); });
    refused("4-byte", [&] { call(s, x, gate, y, first, last, slots, off(lengths, 2), saved, work); });
    refused("16-byte", [&] { call(s, x, gate, y, first, last, slots, lengths, saved + 4, work); });
    refused("requires a workspace", [&] { call(s, x, gate, y, first, last, slots, lengths, saved, nullptr); });

    T *dy = at<T>(10), *dx = at<T>(11), *dgate = at<T>(12);
    const auto back = [&](const thff_scan_shape& shape, T* dy, T* x, T* gate, void* saved, float* dlast, int* lengths,
                          T* dx, T* dgate, float* dfirst, void* work) {
        ThunderFFT_gated_scan_backward<T>(shape, dy, x, gate, saved, dlast, lengths, dx, dgate, dfirst, work);
    };
    refused("another type", [&] { back(ThunderFFT_scan_shape<Other>(2, 300, 70), dy, x, gate, saved, last, lengths, dx, dgate, first, work); });
    refused("alias", [&] { back(s, dy, x, gate, saved, last, lengths, dy, dgate, first, work); });
    refused("alias", [&] { back(s, dy, x, gate, saved, last, lengths, x, dgate, first, work); });
    refused("alias", [&] { back(s, dy, x, gate, saved, last, lengths, dx, gate, first, work); });
    refused("forward call saved", [&] { back(s, dy, x, gate, nullptr, last, lengths, dx, dgate, first, work); });
    refused("4-byte", [&] { back(s, dy, x, gate, saved, off(last, 2), lengths, dx, dgate, first, work); });
    refused("4-byte", [&] { back(s, dy, x, gate, saved, last, off(lengths, 2), dx, dgate, first, work); });
    refused("4-byte", [&] { back(s, dy, x, gate, saved, last, lengths, dx, dgate, off(first, 2), work); });
    refused("requires a workspace", [&] { back(s, dy, x, gate, saved, last, lengths, dx, dgate, first, nullptr); });
}

template <class T>
void norm() {
    T *x = at<T>(1), *y = at<T>(2), *dy = at<T>(3), *dx = at<T>(4);
    float *w = at<float>(5), *b = at<float>(6), *mean = at<float>(7), *rstd = at<float>(8);
    char* work = at<char>(9);
    refused("non-null", [&] { ThunderFFT_layer_norm<T>(nullptr, w, b, 1e-5f, y, 4, 8, mean, rstd); });
    refused("alias", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, x, 4, 8, mean, rstd); });
    refused("eps", [&] { ThunderFFT_layer_norm<T>(x, w, b, -1.0f, y, 4, 8, mean, rstd); });
    refused("cols", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, 4, 0, mean, rstd); });
    refused("rows", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, -4, 8, mean, rstd); });
    refused("4-byte", [&] { ThunderFFT_layer_norm<T>(x, off(w, 2), b, 1e-5f, y, 4, 8, mean, rstd); });
    refused("4-byte", [&] { ThunderFFT_layer_norm<T>(x, w, off(b, 2), 1e-5f, y, 4, 8, mean, rstd); });
    refused("4-byte", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, 4, 8, off(mean, 2), rstd); });
    refused("4-byte", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, 4, 8, mean, off(rstd, 2)); });
    refused("stride", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, 4, 8, mean, rstd, 7); });
    refused("stride", [&] { ThunderFFT_layer_norm<T>(x, w, b, 1e-5f, y, 4, 8, mean, rstd, 8, 7); });
    ThunderFFT_layer_norm<T>(nullptr, nullptr, nullptr, 0.0f, nullptr, 0, 8);  // no rows
    if (ThunderFFT_layer_norm_workspace_bytes(300, 64) != 8 * 256 * 64) std::printf("norm workspace bytes\n");
    refused("rows", [&] { ThunderFFT_layer_norm_workspace_bytes(-1, 64); });
    const auto back = [&](T* dy, T* x, float* mean, float* rstd, float* w, T* dx, float* dw, float* db, void* work,
                          long long dy_stride = 0, long long x_stride = 0, long long dx_stride = 0) {
        ThunderFFT_layer_norm_backward<T>(dy, x, mean, rstd, w, dx, dw, db, work, 4, 8, dy_stride, x_stride, dx_stride);
    };
    float *dw = at<float>(10), *db = at<float>(11);
    refused("alias its inputs", [&] { back(dy, x, mean, rstd, w, dy, dw, db, work); });
    refused("alias its inputs", [&] { back(dy, x, mean, rstd, w, x, dw, db, work); });
    refused("alias dbias", [&] { back(dy, x, mean, rstd, w, dx, dw, dw, work); });
    refused("non-null", [&] { back(dy, x, nullptr, rstd, w, dx, dw, db, work); });
    refused("non-null", [&] { back(dy, x, mean, nullptr, w, dx, dw, db, work); });
    refused("4-byte", [&] { back(dy, x, mean, rstd, off(w, 2), dx, dw, db, work); });
    refused("4-byte", [&] { back(dy, x, mean, rstd, w, dx, off(dw, 2), db, work); });
    refused("4-byte", [&] { back(dy, x, mean, rstd, w, dx, dw, off(db, 2), work); });
    refused("requires a workspace", [&] { back(dy, x, mean, rstd, w, dx, dw, db, nullptr); });
    refused("16-byte", [&] { back(dy, x, mean, rstd, w, dx, dw, db, work + 4); });
    refused("stride", [&] { back(dy, x, mean, rstd, w, dx, dw, db, work, 7); });
    refused("stride", [&] { back(dy, x, mean, rstd, w, dx, dw, db, work, 8, 7); });
    refused("stride", [&] { back(dy, x, mean, rstd, w, dx, dw, db, work, 8, 8, 7); });
}

int main() {
    scan<float, half>();
    scan<half, __hip_bfloat16>();
    scan<__hip_bfloat16, float>();
    norm<float>();
    norm<half>();
    norm<__hip_bfloat16>();
    std::puts("done");
}
"""


def hipcc():
    for cand in (os.environ.get("HIPCC"), os.path.join(ROCM, "bin", "hipcc"), shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    pytest.skip("hipcc not found")


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


@pytest.mark.parametrize("first", ["hip/hip_bf16.h", "thunderfft/thunderfft.hpp"])
def test_templates_compile_beside_the_bfloat16_header(tmp_path, first):
    """With the type's own header before this one or behind it."""
    second = {"hip/hip_bf16.h": "thunderfft/thunderfft.hpp"}.get(first, "hip/hip_bf16.h")
    body = "".join(f"""
template void thunderfft::ThunderFFT_gated_scan<{T}>(const thff_scan_shape&, const {T}*, const {T}*, {T}*, const float*,
    float*, const int*, const int*, void*, void*, hipStream_t);
template void thunderfft::ThunderFFT_gated_scan_backward<{T}>(const thff_scan_shape&, const {T}*, const {T}*, const {T}*,
    const void*, const float*, const int*, {T}*, {T}*, float*, void*, hipStream_t);
template void thunderfft::ThunderFFT_layer_norm<{T}>(const {T}*, const float*, const float*, float, {T}*, long long, int,
    float*, float*, long long, long long, hipStream_t);
template void thunderfft::ThunderFFT_layer_norm_backward<{T}>(const {T}*, const {T}*, const float*, const float*,
    const float*, {T}*, float*, float*, void*, long long, int, long long, long long, long long, hipStream_t);
""" for T in TYPES)
    src = tmp_path / "k.hip"
    src.write_text(f"#include <{first}>\n#include <{second}>\n{body}")
    command = [hipcc(), "--offload-arch=gfx950", "-std=c++17", "-fsyntax-only", "-I", os.path.join(ROOT, "include")]
    res = subprocess.run([*command, str(src)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    src.write_text("#include <thunderfft/thunderfft.hpp>\nauto s = thunderfft::ThunderFFT_scan_shape<double>(1, 1, 1);\n")
    res = subprocess.run([*command, str(src)], capture_output=True, text=True, timeout=300)
    assert res.returncode != 0 and "float, half and __hip_bfloat16 only" in res.stderr
