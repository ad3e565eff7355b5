"""thunderfft_amd -- MI355X (gfx950) ThunderFFT: batched C2C FFTs, N = 64..4096.

Python mirror of the reference's host API (mcrl/thunderfft,
include/thunderfft/thunderfft.cuh:55-63,150-154) over the C ABI of
``libthunderfft_amd.so`` (declared in include/thunderfft/thunderfft.h):

    ThunderFFTInitialize(T, N)                       # T in {"float", "half"}
    ThunderFFT_global(T, N, forward, d_in, d_out, batch, stream=0)
    ThunderFFTFinalize(T)

Errors keep the reference's two kinds: ``ValueError`` where the reference
throws ``std::invalid_argument`` (raised before any HIP call) and
``RuntimeError("[ThunderFFT] ...")`` where it throws ``std::runtime_error``.

Pointers are plain integers (device addresses); torch tensors are accepted
and their ``data_ptr()`` is used.  There is no CPU path: importing this module
fails loudly if the HIP library has not been built.
"""
from __future__ import annotations

import ctypes
import os

__all__ = [
    "SUPPORTED_N", "PRECISIONS", "lib", "ThunderFFTInitialize", "ThunderFFTFinalize",
    "ThunderFFT_global", "ThunderFFT_global_async", "twiddle_info", "fill_uniform",
    "fft", "transforms_per_block", "LIB_PATH", "ThunderFFT_conv1d", "ThunderFFT_conv1d_async",
    "ThunderFFT_conv2d", "ThunderFFT_conv2d_async", "ThunderFFT_conv2d_noalloc", "copy_nt",
    "VALUE_TYPES", "ScanShape", "ThunderFFT_gated_scan", "ThunderFFT_gated_scan_async",
    "ThunderFFT_gated_scan_backward", "ThunderFFT_gated_scan_backward_async",
    "ThunderFFT_layer_norm", "ThunderFFT_layer_norm_async", "ThunderFFT_layer_norm_backward",
    "ThunderFFT_layer_norm_backward_async", "layer_norm_workspace_bytes", "gated_scan",
    "layer_norm", "ConvShape", "ThunderFFT_short_conv", "ThunderFFT_short_conv_async",
    "ThunderFFT_short_conv_backward", "ThunderFFT_short_conv_backward_async", "StateShape",
    "ThunderFFT_state_scan", "ThunderFFT_state_scan_async", "ThunderFFT_state_scan_backward",
    "ThunderFFT_state_scan_backward_async", "ThunderFFT_rms_norm", "ThunderFFT_rms_norm_async",
    "ThunderFFT_rms_norm_8bit", "ThunderFFT_rms_norm_8bit_async", "ThunderFFT_rms_norm_backward",
    "ThunderFFT_rms_norm_backward_async", "rms_norm_workspace_bytes", "short_conv", "state_scan",
    "rms_norm", "rms_norm_8bit",
]

SUPPORTED_N = (64, 128, 256, 512, 1024, 2048, 4096)
PRECISIONS = {"float": 0, "half": 1}
# Types of the sequence operators' values.
VALUE_TYPES = {"float": 0, "half": 1, "bfloat16": 2}
THFF_OK, THFF_EINVAL, THFF_EIO = 0, -22, -5

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libthunderfft_amd.so")

_lib = None
_int32 = None  # torch's, once it is loaded


def lib() -> ctypes.CDLL:
    """Load libthunderfft_amd.so (raises if it has not been built)."""
    global _lib, _int32
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `python -m thunderfft_amd.build` "
                "(there is no CPU fallback)")
        # torch ships its own HIP runtime.  Loaded after this library, it would
        # be a second runtime in the process, and this library's would find no
        # device; loaded first, this library binds to torch's (same soname).
        try:
            import torch

            _int32 = torch.int32
        except ImportError:
            pass
        L = ctypes.CDLL(LIB_PATH)
        vp = ctypes.c_void_p
        L.thff_version.restype = ctypes.c_int
        L.thff_last_error.restype = ctypes.c_char_p
        L.thff_initialize.argtypes = [ctypes.c_int, ctypes.c_int]
        L.thff_finalize.argtypes = [ctypes.c_int]
        sig = [ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, vp, ctypes.c_int, vp]
        L.thff_global.argtypes = sig
        L.thff_global_async.argtypes = sig
        csig = [ctypes.c_int, ctypes.c_int, vp, vp, vp, ctypes.c_int, ctypes.c_int, vp]
        L.thff_conv1d.argtypes = csig
        L.thff_conv1d_async.argtypes = csig
        c2sig = [ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, vp, vp, ctypes.c_int, vp]
        L.thff_conv2d.argtypes = c2sig
        L.thff_conv2d_async.argtypes = c2sig
        L.thff_conv2d_noalloc.argtypes = c2sig
        rfsig = [ctypes.c_int, ctypes.c_int, vp, vp, ctypes.c_int, ctypes.c_float, vp]
        L.thff_conv1d_real_filter.argtypes = rfsig
        L.thff_conv1d_real_filter_async.argtypes = rfsig
        rsig = [ctypes.c_int, ctypes.c_int, vp, vp, vp, ctypes.c_int, ctypes.c_int, vp]
        L.thff_conv1d_real.argtypes = rsig
        L.thff_conv1d_real_async.argtypes = rsig
        vsig = [ctypes.c_int, vp, ctypes.c_longlong, vp, ctypes.c_int, vp, ctypes.c_int, vp]
        L.thff_conv1d_valid.argtypes = vsig
        L.thff_conv1d_valid_async.argtypes = vsig
        L.thff_twiddle_info.argtypes = [ctypes.c_int, ctypes.POINTER(vp),
                                        ctypes.POINTER(ctypes.c_int)]
        L.thff_fill_uniform.argtypes = [ctypes.c_int, vp, ctypes.c_longlong, ctypes.c_ulonglong,
                                        ctypes.c_longlong, vp]
        L.thff_copy_nt.argtypes = [vp, vp, ctypes.c_longlong, vp]
        i32, i64, f32 = ctypes.c_int, ctypes.c_longlong, ctypes.c_float
        sp = ctypes.POINTER(ScanShape)
        for name in ("saved", "workspace"):
            fn = getattr(L, f"thff_gated_scan_{name}_bytes")
            fn.argtypes, fn.restype = [sp], i64
        L.thff_layer_norm_workspace_bytes.argtypes = [i64, i32]
        L.thff_layer_norm_workspace_bytes.restype = i64
        for twin in ("", "_async"):
            getattr(L, "thff_gated_scan" + twin).argtypes = [sp] + [vp] * 10
            getattr(L, "thff_gated_scan_backward" + twin).argtypes = [sp] + [vp] * 11
            getattr(L, "thff_layer_norm" + twin).argtypes = [
                i32, vp, i64, vp, vp, f32, vp, i64, vp, vp, i64, i32, vp]
            getattr(L, "thff_layer_norm_backward" + twin).argtypes = [
                i32, vp, i64, vp, i64, vp, vp, vp, vp, i64, vp, vp, vp, i64, i32, vp]
        cp, tp = ctypes.POINTER(ConvShape), ctypes.POINTER(StateShape)
        for name, p in (("short_conv_workspace", cp), ("state_scan_saved", tp),
                        ("state_scan_forward", tp), ("state_scan_workspace", tp)):
            fn = getattr(L, f"thff_{name}_bytes")
            fn.argtypes, fn.restype = [p], i64
        L.thff_rms_norm_workspace_bytes.argtypes = [i64, i32]
        L.thff_rms_norm_workspace_bytes.restype = i64
        for twin in ("", "_async"):
            getattr(L, "thff_short_conv" + twin).argtypes = [cp] + [vp] * 9
            getattr(L, "thff_short_conv_backward" + twin).argtypes = [cp] + [vp] * 13
            getattr(L, "thff_state_scan" + twin).argtypes = [tp] + [vp] * 16
            getattr(L, "thff_state_scan_backward" + twin).argtypes = [
                tp, ctypes.POINTER(_StateGradients), vp, vp]
            getattr(L, "thff_rms_norm" + twin).argtypes = [
                i32, vp, i64, vp, i64, vp, f32, vp, i64, vp, i64, vp, i64, i32, vp]
            getattr(L, "thff_rms_norm_8bit" + twin).argtypes = [
                i32, vp, i64, vp, i64, vp, f32, vp, i64, vp, i32, vp, i64, i64, i32, vp]
            getattr(L, "thff_rms_norm_backward" + twin).argtypes = [
                i32, vp, i64, vp, i64, vp, vp, vp, i64, vp, i64, vp, vp, i64, i32, vp]
        _lib = L
    return _lib


def _precision(T) -> int:
    if isinstance(T, str) and T in PRECISIONS:
        return PRECISIONS[T]
    name = getattr(T, "__name__", None) or str(T)
    for key, code in (("float16", 1), ("half", 1), ("complex32", 1), ("float32", 0),
                      ("float", 0), ("complex64", 0)):
        if key in name:
            return code
    raise ValueError(f"ThunderFFT supports float and half only (got {T!r})")


def _ptr(x) -> int:
    if x is None:
        return 0
    try:
        return x.data_ptr()
    except AttributeError:
        pass
    if isinstance(x, int):
        return x
    raise TypeError(f"expected a device pointer or tensor, got {type(x).__name__}")


def _ints(x) -> int:
    """_ptr of slots or lengths, which kernels index by: a tensor of them is int32 without gaps, in memory
    that the device reads."""
    if x is None or isinstance(x, int):
        return x or 0
    dtype = getattr(x, "dtype", None)
    if dtype is None:
        return _ptr(x)
    if dtype is not _int32 and str(dtype) != "torch.int32" or not x.is_contiguous():
        raise ValueError(f"slots and lengths must be int32 without gaps (got {dtype}, strides {tuple(x.stride())})")
    if not x.is_cuda and not x.is_pinned():
        raise ValueError("slots and lengths must be in device memory")
    return x.data_ptr()


def _stream(s) -> int:
    if s is None:
        return 0
    if isinstance(s, int):
        return s
    handle = getattr(s, "cuda_stream", None)
    if handle is not None:
        return int(handle)
    if s == 0:
        return 0
    raise TypeError("stream must be an integer hipStream_t or a torch.cuda.Stream")


def _raise(rc: int) -> None:
    if rc == THFF_OK:
        return
    msg = lib().thff_last_error().decode()
    if rc == THFF_EINVAL:
        raise ValueError(msg)
    raise RuntimeError(msg)


def ThunderFFTInitialize(T, N: int) -> None:
    """ThunderFFTInitialize<T>(N): build this device's twiddle table for (T, N)."""
    _raise(lib().thff_initialize(_precision(T), int(N)))


def ThunderFFTFinalize(T) -> None:
    """ThunderFFTFinalize<T>(): release this device's twiddle table for T."""
    _raise(lib().thff_finalize(_precision(T)))


def ThunderFFT_global(T, N: int, forward: bool, d_input, d_output, batch: int, stream=0) -> None:
    """ThunderFFT_global<T,N,forward>(d_input, d_output, batch, stream); synchronous."""
    _raise(lib().thff_global(_precision(T), int(N), int(bool(forward)), _ptr(d_input),
                             _ptr(d_output), int(batch), _stream(stream)))


def ThunderFFT_global_async(T, N: int, forward: bool, d_input, d_output, batch: int,
                            stream=0) -> None:
    """As ThunderFFT_global, but returns once the launch is enqueued on ``stream``."""
    _raise(lib().thff_global_async(_precision(T), int(N), int(bool(forward)), _ptr(d_input),
                                   _ptr(d_output), int(batch), _stream(stream)))


def ThunderFFT_conv1d(T, N: int, d_x, d_h, d_y, batch: int, per_signal_filter: bool = True,
                      stream=0) -> None:
    """Fused circular convolution y[b] = IFFT(FFT(x[b]) * FFT(h[b or 0])) / N; synchronous."""
    _raise(lib().thff_conv1d(_precision(T), int(N), _ptr(d_x), _ptr(d_h), _ptr(d_y), int(batch),
                             int(bool(per_signal_filter)), _stream(stream)))


def ThunderFFT_conv1d_async(T, N: int, d_x, d_h, d_y, batch: int, per_signal_filter: bool = True,
                            stream=0) -> None:
    """As ThunderFFT_conv1d, but returns once the launch is enqueued on ``stream``."""
    _raise(lib().thff_conv1d_async(_precision(T), int(N), _ptr(d_x), _ptr(d_h), _ptr(d_y),
                                   int(batch), int(bool(per_signal_filter)), _stream(stream)))


def ThunderFFT_conv1d_real_filter(T, N: int, d_h, d_spectrum, channels: int, scale: float = 1.0,
                                  stream=0) -> None:
    """spectrum[d] = scale * FFT(h[d]) for real fp32 filters h (channels, N) -> complex64
    spectra (channels, N), for ThunderFFT_conv1d_real of type T; synchronous."""
    _raise(lib().thff_conv1d_real_filter(_precision(T), int(N), _ptr(d_h), _ptr(d_spectrum),
                                         int(channels), float(scale), _stream(stream)))


def ThunderFFT_conv1d_real_filter_async(T, N: int, d_h, d_spectrum, channels: int,
                                        scale: float = 1.0, stream=0) -> None:
    """As ThunderFFT_conv1d_real_filter, but returns once the launch is enqueued."""
    _raise(lib().thff_conv1d_real_filter_async(_precision(T), int(N), _ptr(d_h), _ptr(d_spectrum),
                                               int(channels), float(scale), _stream(stream)))


def ThunderFFT_conv1d_real(T, N: int, d_x, d_spectrum, d_y, batch: int, channels: int,
                           stream=0) -> None:
    """Real fused convolution y[b][d] = Re IFFT(FFT(x[b][d]) * spectrum[d]) of real
    (batch, channels, N) signals of type T; synchronous."""
    _raise(lib().thff_conv1d_real(_precision(T), int(N), _ptr(d_x), _ptr(d_spectrum), _ptr(d_y),
                                  int(batch), int(channels), _stream(stream)))


def ThunderFFT_conv1d_real_async(T, N: int, d_x, d_spectrum, d_y, batch: int, channels: int,
                                 stream=0) -> None:
    """As ThunderFFT_conv1d_real, but returns once the launch is enqueued on ``stream``."""
    _raise(lib().thff_conv1d_real_async(_precision(T), int(N), _ptr(d_x), _ptr(d_spectrum),
                                        _ptr(d_y), int(batch), int(channels), _stream(stream)))


def ThunderFFT_conv1d_valid(T, d_x, input_len: int, d_taps, filter_len: int, d_y, batch: int = 1,
                            stream=0) -> None:
    """Valid correlation y[b][i] = sum_k x[b][i + k] * taps[k] (complex, type T; taps
    complex64, 1 <= filter_len <= 64); needs the table of N = 64; synchronous."""
    _raise(lib().thff_conv1d_valid(_precision(T), _ptr(d_x), int(input_len), _ptr(d_taps),
                                   int(filter_len), _ptr(d_y), int(batch), _stream(stream)))


def ThunderFFT_conv1d_valid_async(T, d_x, input_len: int, d_taps, filter_len: int, d_y,
                                  batch: int = 1, stream=0) -> None:
    """As ThunderFFT_conv1d_valid, but returns once the launch is enqueued on ``stream``."""
    _raise(lib().thff_conv1d_valid_async(_precision(T), _ptr(d_x), int(input_len), _ptr(d_taps),
                                         int(filter_len), _ptr(d_y), int(batch), _stream(stream)))


def ThunderFFT_conv2d(T, rows: int, cols: int, d_x, d_h, d_y, batch: int, stream=0) -> None:
    """2-D circular convolution y[b] = IFFT2(FFT2(x[b]) * FFT2(h)) / (rows*cols) with
    one shared filter: 64 x 64 and 128 x 128 images in one fused kernel per image,
    1024 x 1024 as row pass, fused column pass, inverse row pass; synchronous."""
    _raise(lib().thff_conv2d(_precision(T), int(rows), int(cols), _ptr(d_x), _ptr(d_h), _ptr(d_y),
                             int(batch), _stream(stream)))


def ThunderFFT_conv2d_async(T, rows: int, cols: int, d_x, d_h, d_y, batch: int, stream=0) -> None:
    """As ThunderFFT_conv2d, but returns once the launch is enqueued on ``stream``."""
    _raise(lib().thff_conv2d_async(_precision(T), int(rows), int(cols), _ptr(d_x), _ptr(d_h),
                                   _ptr(d_y), int(batch), _stream(stream)))


def ThunderFFT_conv2d_noalloc(T, rows: int, cols: int, d_x, d_h, d_y, batch: int,
                              stream=0) -> None:
    """As ThunderFFT_conv2d_async, but allocates no device memory (the 1024 x 1024
    form keeps its filter spectrum in the library's per-GPU device array; calls
    that overlap on one GPU race)."""
    _raise(lib().thff_conv2d_noalloc(_precision(T), int(rows), int(cols), _ptr(d_x), _ptr(d_h),
                                     _ptr(d_y), int(batch), _stream(stream)))


def _value_type(T) -> int:
    code = VALUE_TYPES.get(T) if isinstance(T, str) else None
    if code is not None:
        return code
    name = str(T).rpartition(".")[2]
    for key, code in (("float32", 0), ("float16", 1), ("bfloat16", 2)):
        if name == key:
            return code
    raise ValueError(f"the sequence operators support float, half and bfloat16 only (got {T!r})")


class ScanShape(ctypes.Structure):
    """What a gated scan works on; kept by the caller from call to call.

    T: "float", "half" or "bfloat16" (or the torch dtype).  layout: "channels_last",
    values [batch][n][channels], or "channels_first", values [batch][channels][n] as the
    convolutions have them.  Strides: elements between the starts of consecutive rows (a
    step's channels, or a channel's steps), None for rows without a gap; x_stride and
    gate_stride hold for the gradients of x and the gate too.  states: rows of the state
    pool that slots index (None: batch).
    """

    _fields_ = [("precision", ctypes.c_int), ("layout", ctypes.c_int), ("batch", ctypes.c_int),
                ("n", ctypes.c_int), ("channels", ctypes.c_int), ("states", ctypes.c_int),
                ("x_stride", ctypes.c_longlong), ("gate_stride", ctypes.c_longlong),
                ("y_stride", ctypes.c_longlong)]
    LAYOUTS = {"channels_last": 0, "channels_first": 1}

    def __init__(self, T, batch, n, channels, layout="channels_last", x_stride=None,
                 gate_stride=None, y_stride=None, states=None):
        if layout not in self.LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(self.LAYOUTS)} (got {layout!r})")
        states = batch if states is None else states
        for v, what in ((batch, "batch"), (n, "n"), (channels, "channels"), (states, "states")):
            if not -2**31 <= int(v) < 2**31:
                raise ValueError(f"{what} is out of range")
        super().__init__(_value_type(T), self.LAYOUTS[layout], int(batch), int(n), int(channels),
                         int(states), int(x_stride or 0), int(gate_stride or 0),
                         int(y_stride or 0))

    def saved_bytes(self) -> int:
        """Bytes that the forward call keeps for the backward call (d_saved)."""
        return _bytes(lib().thff_gated_scan_saved_bytes(ctypes.byref(self)))

    def workspace_bytes(self) -> int:
        """Bytes of a call's scratch memory (d_workspace)."""
        return _bytes(lib().thff_gated_scan_workspace_bytes(ctypes.byref(self)))


def _bytes(rc: int) -> int:
    if rc < 0:
        _raise(int(rc))
    return int(rc)


def _gated_scan(call, shape, d_x, d_gate, d_y, d_state_in, d_state_out, d_slots, d_lengths,
                d_saved, d_workspace, stream):
    _raise(call(shape, _ptr(d_x), _ptr(d_gate), _ptr(d_y), _ptr(d_state_in), _ptr(d_state_out),
                _ints(d_slots), _ints(d_lengths), _ptr(d_saved), _ptr(d_workspace), _stream(stream)))


def ThunderFFT_gated_scan(shape, d_x, d_gate, d_y, d_state_in=None, d_state_out=None, d_slots=None,
                          d_lengths=None, d_saved=None, d_workspace=None, stream=0) -> None:
    """Gated linear recurrence h[t] = f[t] h[t-1] + (1 - f[t]) x[t], f = sigmoid(gate), y = h,
    on values of ``shape`` (a ScanShape).  The states before the first step (d_state_in) and
    after the last (d_state_out, the same buffer if wanted) are float32 rows of `channels`,
    row b for sequence b or row d_slots[b] (int32) of a pool; d_lengths (int32) ends each
    sequence early.  d_saved (shape.saved_bytes()) is kept for the backward call, d_workspace
    (shape.workspace_bytes()) is scratch.  Synchronous."""
    _gated_scan(lib().thff_gated_scan, shape, d_x, d_gate, d_y, d_state_in, d_state_out, d_slots,
                d_lengths, d_saved, d_workspace, stream)


def ThunderFFT_gated_scan_async(shape, d_x, d_gate, d_y, d_state_in=None, d_state_out=None,
                                d_slots=None, d_lengths=None, d_saved=None, d_workspace=None,
                                stream=0) -> None:
    """As ThunderFFT_gated_scan, but returns once the work is enqueued on ``stream``."""
    _gated_scan(lib().thff_gated_scan_async, shape, d_x, d_gate, d_y, d_state_in, d_state_out,
                d_slots, d_lengths, d_saved, d_workspace, stream)


def _gated_scan_backward(call, shape, d_dy, d_x, d_gate, d_saved, d_dx, d_dgate, d_dstate_out,
                         d_dstate_in, d_lengths, d_workspace, stream):
    _raise(call(shape, _ptr(d_dy), _ptr(d_x), _ptr(d_gate), _ptr(d_saved), _ptr(d_dstate_out),
                _ints(d_lengths), _ptr(d_dx), _ptr(d_dgate), _ptr(d_dstate_in), _ptr(d_workspace),
                _stream(stream)))


def ThunderFFT_gated_scan_backward(shape, d_dy, d_x, d_gate, d_saved, d_dx, d_dgate,
                                   d_dstate_out=None, d_dstate_in=None, d_lengths=None,
                                   d_workspace=None, stream=0) -> None:
    """Gradients of ThunderFFT_gated_scan by x, the gate and the first state (d_dstate_in,
    float32 [batch][channels]) from those by y (d_dy) and by the last states (d_dstate_out,
    None: zero); d_saved is what the forward call of the same shape, x, gate and lengths
    wrote.  Synchronous."""
    _gated_scan_backward(lib().thff_gated_scan_backward, shape, d_dy, d_x, d_gate, d_saved, d_dx,
                         d_dgate, d_dstate_out, d_dstate_in, d_lengths, d_workspace, stream)


def ThunderFFT_gated_scan_backward_async(shape, d_dy, d_x, d_gate, d_saved, d_dx, d_dgate,
                                         d_dstate_out=None, d_dstate_in=None, d_lengths=None,
                                         d_workspace=None, stream=0) -> None:
    """As ThunderFFT_gated_scan_backward, but returns once the work is enqueued."""
    _gated_scan_backward(lib().thff_gated_scan_backward_async, shape, d_dy, d_x, d_gate, d_saved,
                         d_dx, d_dgate, d_dstate_out, d_dstate_in, d_lengths, d_workspace, stream)


def _layer_norm(call, T, d_x, d_weight, d_bias, eps, d_y, rows, cols, d_mean, d_rstd, x_stride,
                y_stride, stream):
    _raise(call(_value_type(T), _ptr(d_x), x_stride or 0, _ptr(d_weight), _ptr(d_bias), eps,
                _ptr(d_y), y_stride or 0, _ptr(d_mean), _ptr(d_rstd), rows, _int(cols),
                _stream(stream)))


def _int(v) -> int:
    # ctypes would wrap a larger number round.
    if not -2**31 <= v < 2**31:
        raise ValueError(f"{v} is out of range")
    return v


def ThunderFFT_layer_norm(T, d_x, d_weight, d_bias, eps, d_y, rows, cols, d_mean=None, d_rstd=None,
                          x_stride=None, y_stride=None, stream=0) -> None:
    """Layer norm y = (x - mean) rstd weight + bias of `rows` rows of `cols` values of type T;
    weight and bias float32 (None: ones, zeros); d_mean and d_rstd (float32, one a row) keep
    the statistics for the backward call.  Synchronous."""
    _layer_norm(lib().thff_layer_norm, T, d_x, d_weight, d_bias, eps, d_y, rows, cols, d_mean,
                d_rstd, x_stride, y_stride, stream)


def ThunderFFT_layer_norm_async(T, d_x, d_weight, d_bias, eps, d_y, rows, cols, d_mean=None,
                                d_rstd=None, x_stride=None, y_stride=None, stream=0) -> None:
    """As ThunderFFT_layer_norm, but returns once the launch is enqueued on ``stream``."""
    _layer_norm(lib().thff_layer_norm_async, T, d_x, d_weight, d_bias, eps, d_y, rows, cols, d_mean,
                d_rstd, x_stride, y_stride, stream)


def layer_norm_workspace_bytes(rows: int, cols: int) -> int:
    """Bytes of ThunderFFT_layer_norm_backward's d_workspace."""
    return _bytes(lib().thff_layer_norm_workspace_bytes(int(rows), _int(int(cols))))


def _layer_norm_backward(call, T, d_dy, d_x, d_mean, d_rstd, d_weight, d_dx, d_dweight, d_dbias,
                         d_workspace, rows, cols, dy_stride, x_stride, dx_stride, stream):
    _raise(call(_value_type(T), _ptr(d_dy), dy_stride or 0, _ptr(d_x), x_stride or 0, _ptr(d_mean),
                _ptr(d_rstd), _ptr(d_weight), _ptr(d_dx), dx_stride or 0, _ptr(d_dweight),
                _ptr(d_dbias), _ptr(d_workspace), rows, _int(cols), _stream(stream)))


def ThunderFFT_layer_norm_backward(T, d_dy, d_x, d_mean, d_rstd, d_weight, d_dx, d_dweight, d_dbias,
                                   d_workspace, rows, cols, dy_stride=None, x_stride=None,
                                   dx_stride=None, stream=0) -> None:
    """Gradients of ThunderFFT_layer_norm by x and, in float32, by the weight and the bias
    (None: not computed), from that by y, x and the forward call's statistics.  Synchronous."""
    _layer_norm_backward(lib().thff_layer_norm_backward, T, d_dy, d_x, d_mean, d_rstd, d_weight,
                         d_dx, d_dweight, d_dbias, d_workspace, rows, cols, dy_stride, x_stride,
                         dx_stride, stream)


def ThunderFFT_layer_norm_backward_async(T, d_dy, d_x, d_mean, d_rstd, d_weight, d_dx, d_dweight,
                                         d_dbias, d_workspace, rows, cols, dy_stride=None,
                                         x_stride=None, dx_stride=None, stream=0) -> None:
    """As ThunderFFT_layer_norm_backward, but returns once the work is enqueued."""
    _layer_norm_backward(lib().thff_layer_norm_backward_async, T, d_dy, d_x, d_mean, d_rstd,
                         d_weight, d_dx, d_dweight, d_dbias, d_workspace, rows, cols, dy_stride,
                         x_stride, dx_stride, stream)


def _sizes(**named):
    """The values as integers; ctypes would wrap larger ones round."""
    for what, v in named.items():
        if not -2**31 <= int(v) < 2**31:
            raise ValueError(f"{what} is out of range")
    return [int(v) for v in named.values()]


class ConvShape(ctypes.Structure):
    """What a short convolution works on; kept by the caller from call to call.

    T: "float", "half" or "bfloat16" (or the torch dtype), of values [batch][n][channels].
    width: taps, 2 to 4.  silu: whether the activation follows.  Strides: elements between the
    starts of consecutive rows, None for rows without a gap; each holds for its array's
    gradient too.  states: rows of the state pool that slots index (None: batch).
    """

    _fields_ = [("precision", ctypes.c_int), ("silu", ctypes.c_int), ("batch", ctypes.c_int),
                ("n", ctypes.c_int), ("channels", ctypes.c_int), ("width", ctypes.c_int),
                ("states", ctypes.c_int), ("x_stride", ctypes.c_longlong),
                ("y_stride", ctypes.c_longlong)]

    def __init__(self, T, batch, n, channels, width, silu=True, x_stride=None, y_stride=None,
                 states=None):
        sizes = _sizes(batch=batch, n=n, channels=channels, width=width,
                       states=batch if states is None else states)
        super().__init__(_value_type(T), int(bool(silu)), *sizes, int(x_stride or 0),
                         int(y_stride or 0))

    def workspace_bytes(self) -> int:
        """Bytes of a backward call's scratch memory (d_workspace)."""
        return _bytes(lib().thff_short_conv_workspace_bytes(ctypes.byref(self)))


def _short_conv(call, shape, d_x, d_weight, d_bias, d_y, d_state_in, d_state_out, d_slots, d_lengths,
                stream):
    _raise(call(shape, _ptr(d_x), _ptr(d_weight), _ptr(d_bias), _ptr(d_y), _ptr(d_state_in),
                _ptr(d_state_out), _ints(d_slots), _ints(d_lengths), _stream(stream)))


def ThunderFFT_short_conv(shape, d_x, d_weight, d_bias, d_y, d_state_in=None, d_state_out=None,
                          d_slots=None, d_lengths=None, stream=0) -> None:
    """Short causal convolution y[t] = silu(bias + sum_k weight[k] x[t - width + 1 + k]) of each
    channel, on values of ``shape`` (a ConvShape); weight float32 [channels][width], bias float32
    [channels] (None: zeros).  The width - 1 values before the first step (d_state_in) and the last
    ones (d_state_out, the same buffer if wanted) are rows [width - 1][channels] of the shape's type,
    row b for sequence b or row d_slots[b] (int32) of a pool; d_lengths (int32) ends each sequence
    early.  Synchronous."""
    _short_conv(lib().thff_short_conv, shape, d_x, d_weight, d_bias, d_y, d_state_in, d_state_out,
                d_slots, d_lengths, stream)


def ThunderFFT_short_conv_async(shape, d_x, d_weight, d_bias, d_y, d_state_in=None,
                                d_state_out=None, d_slots=None, d_lengths=None, stream=0) -> None:
    """As ThunderFFT_short_conv, but returns once the work is enqueued on ``stream``."""
    _short_conv(lib().thff_short_conv_async, shape, d_x, d_weight, d_bias, d_y, d_state_in,
                d_state_out, d_slots, d_lengths, stream)


def _short_conv_backward(call, shape, d_dy, d_x, d_weight, d_bias, d_dx, d_dweight, d_dbias,
                         d_state_in, d_dstate_out, d_dstate_in, d_lengths, d_workspace, stream):
    _raise(call(shape, _ptr(d_dy), _ptr(d_x), _ptr(d_weight), _ptr(d_bias), _ptr(d_state_in),
                _ptr(d_dstate_out), _ints(d_lengths), _ptr(d_dx), _ptr(d_dweight), _ptr(d_dbias),
                _ptr(d_dstate_in), _ptr(d_workspace), _stream(stream)))


def ThunderFFT_short_conv_backward(shape, d_dy, d_x, d_weight, d_bias, d_dx, d_dweight=None,
                                   d_dbias=None, d_state_in=None, d_dstate_out=None,
                                   d_dstate_in=None, d_lengths=None, d_workspace=None,
                                   stream=0) -> None:
    """Gradients of ThunderFFT_short_conv by x, by the weights and the bias (float32; None: not
    computed) and by the first state (d_dstate_in), from those by y and by the last states
    (d_dstate_out, None: zero); states and their gradients are row b for sequence b, of the shape's
    type.  d_workspace: shape.workspace_bytes().  Synchronous."""
    _short_conv_backward(lib().thff_short_conv_backward, shape, d_dy, d_x, d_weight, d_bias, d_dx,
                         d_dweight, d_dbias, d_state_in, d_dstate_out, d_dstate_in, d_lengths,
                         d_workspace, stream)


def ThunderFFT_short_conv_backward_async(shape, d_dy, d_x, d_weight, d_bias, d_dx, d_dweight=None,
                                         d_dbias=None, d_state_in=None, d_dstate_out=None,
                                         d_dstate_in=None, d_lengths=None, d_workspace=None,
                                         stream=0) -> None:
    """As ThunderFFT_short_conv_backward, but returns once the work is enqueued."""
    _short_conv_backward(lib().thff_short_conv_backward_async, shape, d_dy, d_x, d_weight, d_bias,
                         d_dx, d_dweight, d_dbias, d_state_in, d_dstate_out, d_dstate_in,
                         d_lengths, d_workspace, stream)


class StateShape(ctypes.Structure):
    """What a state space scan works on; kept by the caller from call to call.

    T: "float", "half" or "bfloat16" (or the torch dtype), of x, delta, the gate and y,
    [batch][n][channels], and of b and c, [batch][n][groups][order].  order: states of a channel, 1
    to 64.  groups divide the channels.  Strides: elements between the starts of consecutive rows,
    None for rows without a gap; each holds for its array's gradient too.  states: rows of the state
    pool that slots index (None: batch).
    """

    _fields_ = [("precision", ctypes.c_int), ("batch", ctypes.c_int), ("n", ctypes.c_int),
                ("channels", ctypes.c_int), ("order", ctypes.c_int), ("groups", ctypes.c_int),
                ("states", ctypes.c_int), ("x_stride", ctypes.c_longlong),
                ("delta_stride", ctypes.c_longlong), ("gate_stride", ctypes.c_longlong),
                ("b_stride", ctypes.c_longlong), ("c_stride", ctypes.c_longlong),
                ("y_stride", ctypes.c_longlong)]

    def __init__(self, T, batch, n, channels, order, groups=1, x_stride=None, delta_stride=None,
                 gate_stride=None, b_stride=None, c_stride=None, y_stride=None, states=None):
        sizes = _sizes(batch=batch, n=n, channels=channels, order=order, groups=groups,
                       states=batch if states is None else states)
        super().__init__(_value_type(T), *sizes,
                         *(int(v or 0) for v in (x_stride, delta_stride, gate_stride, b_stride,
                                                 c_stride, y_stride)))

    def saved_bytes(self) -> int:
        """Bytes that the forward call keeps for the backward call (d_saved)."""
        return _bytes(lib().thff_state_scan_saved_bytes(ctypes.byref(self)))

    def forward_bytes(self) -> int:
        """Bytes of a forward call's scratch memory alone."""
        return _bytes(lib().thff_state_scan_forward_bytes(ctypes.byref(self)))

    def workspace_bytes(self) -> int:
        """Bytes of a call's scratch memory (d_workspace), enough for forward and backward calls."""
        return _bytes(lib().thff_state_scan_workspace_bytes(ctypes.byref(self)))


def _state_scan(call, shape, d_x, d_delta, d_a, d_b, d_c, d_y, d_skip, d_gate, d_delta_bias, d_state_in,
                d_state_out, d_slots, d_lengths, d_saved, d_workspace, stream):
    _raise(call(shape, _ptr(d_x), _ptr(d_delta), _ptr(d_a), _ptr(d_b), _ptr(d_c), _ptr(d_skip),
                _ptr(d_gate), _ptr(d_delta_bias), _ptr(d_y), _ptr(d_state_in), _ptr(d_state_out),
                _ints(d_slots), _ints(d_lengths), _ptr(d_saved), _ptr(d_workspace), _stream(stream)))


def ThunderFFT_state_scan(shape, d_x, d_delta, d_a, d_b, d_c, d_y, d_skip=None, d_gate=None,
                          d_delta_bias=None, d_state_in=None, d_state_out=None, d_slots=None,
                          d_lengths=None, d_saved=None, d_workspace=None, stream=0) -> None:
    """State space scan on values of ``shape`` (a StateShape): dt = softplus(delta + delta_bias),
    h[t] = exp(dt a) h[t-1] + dt x b for each of a channel's states, y = (sum of c h + skip x)
    silu(gate).  a is float32 [channels][order], skip and delta_bias float32 [channels] (None:
    zeros); without a gate y is the sum.  The states before the first step (d_state_in) and after
    the last (d_state_out, the same buffer if wanted) are float32 rows [channels][order], row b for
    sequence b or row d_slots[b] (int32) of a pool; d_lengths (int32) ends each sequence early.
    d_saved (shape.saved_bytes()) is kept for the backward call, d_workspace
    (shape.forward_bytes()) is scratch.  Synchronous."""
    _state_scan(lib().thff_state_scan, shape, d_x, d_delta, d_a, d_b, d_c, d_y, d_skip, d_gate,
                d_delta_bias, d_state_in, d_state_out, d_slots, d_lengths, d_saved, d_workspace,
                stream)


def ThunderFFT_state_scan_async(shape, d_x, d_delta, d_a, d_b, d_c, d_y, d_skip=None, d_gate=None,
                                d_delta_bias=None, d_state_in=None, d_state_out=None, d_slots=None,
                                d_lengths=None, d_saved=None, d_workspace=None, stream=0) -> None:
    """As ThunderFFT_state_scan, but returns once the work is enqueued on ``stream``."""
    _state_scan(lib().thff_state_scan_async, shape, d_x, d_delta, d_a, d_b, d_c, d_y, d_skip, d_gate,
                d_delta_bias, d_state_in, d_state_out, d_slots, d_lengths, d_saved, d_workspace,
                stream)


class _StateGradients(ctypes.Structure):
    """thff_state_gradients: the arrays of a backward call."""

    _fields_ = [(name, ctypes.c_void_p) for name in (
        "dy", "x", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "saved", "dstate_out",
        "lengths", "dx", "ddelta", "da", "db", "dc", "dskip", "dgate", "ddelta_bias", "dstate_in")]


def _state_scan_backward(call, shape, d_dy, d_x, d_delta, d_a, d_b, d_c, d_saved, d_dx, d_ddelta, d_da,
                         d_db, d_dc, d_skip, d_dskip, d_gate, d_dgate, d_delta_bias, d_ddelta_bias,
                         d_dstate_out, d_dstate_in, d_lengths, d_workspace, stream):
    arrays = _StateGradients(*map(_ptr, (
        d_dy, d_x, d_delta, d_a, d_b, d_c, d_skip, d_gate, d_delta_bias, d_saved, d_dstate_out,
        _ints(d_lengths), d_dx, d_ddelta, d_da, d_db, d_dc, d_dskip, d_dgate, d_ddelta_bias, d_dstate_in)))
    _raise(call(shape, arrays, _ptr(d_workspace), _stream(stream)))


def ThunderFFT_state_scan_backward(shape, d_dy, d_x, d_delta, d_a, d_b, d_c, d_saved, d_dx, d_ddelta,
                                   d_da, d_db, d_dc, d_skip=None, d_dskip=None, d_gate=None,
                                   d_dgate=None, d_delta_bias=None, d_ddelta_bias=None,
                                   d_dstate_out=None, d_dstate_in=None, d_lengths=None,
                                   d_workspace=None, stream=0) -> None:
    """Gradients of ThunderFFT_state_scan from those by y (d_dy) and by the last states
    (d_dstate_out, None: zero), by x, delta, b, c and the gate (d_dgate, where there is one) in the
    shape's type, and by a, skip, the bias (the latter two None: not computed) and the first state
    (None: not stored) in float32.  d_saved is what the forward call of the same shape and inputs
    wrote.  Synchronous."""
    _state_scan_backward(lib().thff_state_scan_backward, shape, d_dy, d_x, d_delta, d_a, d_b, d_c,
                         d_saved, d_dx, d_ddelta, d_da, d_db, d_dc, d_skip, d_dskip, d_gate, d_dgate,
                         d_delta_bias, d_ddelta_bias, d_dstate_out, d_dstate_in, d_lengths,
                         d_workspace, stream)


def ThunderFFT_state_scan_backward_async(shape, d_dy, d_x, d_delta, d_a, d_b, d_c, d_saved, d_dx,
                                         d_ddelta, d_da, d_db, d_dc, d_skip=None, d_dskip=None,
                                         d_gate=None, d_dgate=None, d_delta_bias=None,
                                         d_ddelta_bias=None, d_dstate_out=None, d_dstate_in=None,
                                         d_lengths=None, d_workspace=None, stream=0) -> None:
    """As ThunderFFT_state_scan_backward, but returns once the work is enqueued."""
    _state_scan_backward(lib().thff_state_scan_backward_async, shape, d_dy, d_x, d_delta, d_a, d_b,
                         d_c, d_saved, d_dx, d_ddelta, d_da, d_db, d_dc, d_skip, d_dskip, d_gate,
                         d_dgate, d_delta_bias, d_ddelta_bias, d_dstate_out, d_dstate_in, d_lengths,
                         d_workspace, stream)


def _rms_norm(call, T, d_x, d_weight, eps, d_y, rows, cols, d_residual, d_sum, d_rstd, x_stride,
              residual_stride, y_stride, sum_stride, stream):
    _raise(call(_value_type(T), _ptr(d_x), x_stride or 0, _ptr(d_residual), residual_stride or 0,
                _ptr(d_weight), eps, _ptr(d_y), y_stride or 0, _ptr(d_sum), sum_stride or 0,
                _ptr(d_rstd), rows, _int(cols), _stream(stream)))


def ThunderFFT_rms_norm(T, d_x, d_weight, eps, d_y, rows, cols, d_residual=None, d_sum=None,
                        d_rstd=None, x_stride=None, residual_stride=None, y_stride=None,
                        sum_stride=None, stream=0) -> None:
    """Root-mean-square norm y = s rstd weight of `rows` rows of `cols` values of type T, with
    s = x + d_residual rounded to T (None: s = x), which goes to d_sum (the residual's own buffer if
    wanted; None: not stored); weight float32 (None: ones); d_rstd (float32, one a row) keeps the
    statistics for the backward call.  Synchronous."""
    _rms_norm(lib().thff_rms_norm, T, d_x, d_weight, eps, d_y, rows, cols, d_residual, d_sum, d_rstd,
              x_stride, residual_stride, y_stride, sum_stride, stream)


def ThunderFFT_rms_norm_async(T, d_x, d_weight, eps, d_y, rows, cols, d_residual=None, d_sum=None,
                              d_rstd=None, x_stride=None, residual_stride=None, y_stride=None,
                              sum_stride=None, stream=0) -> None:
    """As ThunderFFT_rms_norm, but returns once the launch is enqueued on ``stream``."""
    _rms_norm(lib().thff_rms_norm_async, T, d_x, d_weight, eps, d_y, rows, cols, d_residual, d_sum,
              d_rstd, x_stride, residual_stride, y_stride, sum_stride, stream)


def _rms_norm_8bit(call, T, d_x, d_weight, eps, d_q, d_scales, rows, cols, block, d_residual, d_sum,
                   x_stride, residual_stride, q_stride, sum_stride, stream):
    _raise(call(_value_type(T), _ptr(d_x), x_stride or 0, _ptr(d_residual), residual_stride or 0,
                _ptr(d_weight), eps, _ptr(d_q), q_stride or 0, _ptr(d_scales), _int(block),
                _ptr(d_sum), sum_stride or 0, rows, _int(cols), _stream(stream)))


def ThunderFFT_rms_norm_8bit(T, d_x, d_weight, eps, d_q, d_scales, rows, cols, block=128,
                             d_residual=None, d_sum=None, x_stride=None, residual_stride=None,
                             q_stride=None, sum_stride=None, stream=0) -> None:
    """As ThunderFFT_rms_norm, with an output of 8 bits (e4m3, torch.float8_e4m3fn) and a float32
    scale for every `block` columns of a row (128, or cols): y is near d_q * scale, the scale the
    largest |y| of the block / 448.  Synchronous."""
    _rms_norm_8bit(lib().thff_rms_norm_8bit, T, d_x, d_weight, eps, d_q, d_scales, rows, cols, block,
                   d_residual, d_sum, x_stride, residual_stride, q_stride, sum_stride, stream)


def ThunderFFT_rms_norm_8bit_async(T, d_x, d_weight, eps, d_q, d_scales, rows, cols, block=128,
                                   d_residual=None, d_sum=None, x_stride=None, residual_stride=None,
                                   q_stride=None, sum_stride=None, stream=0) -> None:
    """As ThunderFFT_rms_norm_8bit, but returns once the launch is enqueued on ``stream``."""
    _rms_norm_8bit(lib().thff_rms_norm_8bit_async, T, d_x, d_weight, eps, d_q, d_scales, rows, cols,
                   block, d_residual, d_sum, x_stride, residual_stride, q_stride, sum_stride, stream)


def rms_norm_workspace_bytes(rows: int, cols: int) -> int:
    """Bytes of ThunderFFT_rms_norm_backward's d_workspace."""
    return _bytes(lib().thff_rms_norm_workspace_bytes(int(rows), _int(int(cols))))


def _rms_norm_backward(call, T, d_dy, d_sum, d_rstd, d_weight, d_dx, d_dweight, d_workspace, rows, cols,
                       d_dsum, dy_stride, sum_stride, dsum_stride, dx_stride, stream):
    _raise(call(_value_type(T), _ptr(d_dy), dy_stride or 0, _ptr(d_sum), sum_stride or 0, _ptr(d_rstd),
                _ptr(d_weight), _ptr(d_dsum), dsum_stride or 0, _ptr(d_dx), dx_stride or 0,
                _ptr(d_dweight), _ptr(d_workspace), rows, _int(cols), _stream(stream)))


def ThunderFFT_rms_norm_backward(T, d_dy, d_sum, d_rstd, d_weight, d_dx, d_dweight, d_workspace, rows,
                                 cols, d_dsum=None, dy_stride=None, sum_stride=None, dsum_stride=None,
                                 dx_stride=None, stream=0) -> None:
    """Gradients of ThunderFFT_rms_norm by x (the residual's is the same) and, in float32, by the
    weight (None: not computed), from that by y (d_dy), the one that reaches the sums from elsewhere
    (d_dsum, None: zero), the sums (x itself without a residual) and the forward call's statistics.
    Synchronous."""
    _rms_norm_backward(lib().thff_rms_norm_backward, T, d_dy, d_sum, d_rstd, d_weight, d_dx, d_dweight,
                       d_workspace, rows, cols, d_dsum, dy_stride, sum_stride, dsum_stride, dx_stride,
                       stream)


def ThunderFFT_rms_norm_backward_async(T, d_dy, d_sum, d_rstd, d_weight, d_dx, d_dweight, d_workspace,
                                       rows, cols, d_dsum=None, dy_stride=None, sum_stride=None,
                                       dsum_stride=None, dx_stride=None, stream=0) -> None:
    """As ThunderFFT_rms_norm_backward, but returns once the work is enqueued."""
    _rms_norm_backward(lib().thff_rms_norm_backward_async, T, d_dy, d_sum, d_rstd, d_weight, d_dx,
                       d_dweight, d_workspace, rows, cols, d_dsum, dy_stride, sum_stride, dsum_stride,
                       dx_stride, stream)


def gated_scan(x, gate, state=None, lengths=None, layout="channels_last"):
    """(y, last states) of the gated linear recurrence on CUDA tensors, differentiable by x,
    gate and state: see thunderfft_amd.sequence.gated_scan."""
    from . import sequence

    return sequence.gated_scan(x, gate, state, lengths, layout)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Layer norm of a CUDA tensor's last axis, differentiable by x, weight and bias: see
    thunderfft_amd.sequence.layer_norm."""
    from . import sequence

    return sequence.layer_norm(x, weight, bias, eps)


def short_conv(x, weight, bias=None, state=None, lengths=None, silu: bool = True):
    """(y, last state) of the short causal convolution on CUDA tensors, differentiable by x, weight,
    bias and state: see thunderfft_amd.block.short_conv."""
    from . import block

    return block.short_conv(x, weight, bias, state, lengths, silu)


def state_scan(x, delta, a, b, c, skip=None, gate=None, delta_bias=None, state=None, lengths=None):
    """(y, last states) of the state space scan on CUDA tensors, differentiable by all its floating
    arguments: see thunderfft_amd.block.state_scan."""
    from . import block

    return block.state_scan(x, delta, a, b, c, skip, gate, delta_bias, state, lengths)


def rms_norm(x, weight=None, residual=None, eps: float = 1e-5):
    """Root-mean-square norm of a CUDA tensor's last axis, with a residual (y, x + residual),
    differentiable by x, weight and residual: see thunderfft_amd.block.rms_norm."""
    from . import block

    return block.rms_norm(x, weight, residual, eps)


def rms_norm_8bit(x, weight=None, residual=None, eps: float = 1e-5, block: int | None = 128):
    """(q, scales) of the norm in 8 bits, with a residual (q, scales, x + residual): see
    thunderfft_amd.block.rms_norm_8bit."""
    from . import block as operators

    return operators.rms_norm_8bit(x, weight, residual, eps, block)


def twiddle_info(T) -> tuple[int, int]:
    """(device pointer, N) of this device's twiddle table for T; (0, 0) when released."""
    p = ctypes.c_void_p()
    n = ctypes.c_int()
    _raise(lib().thff_twiddle_info(_precision(T), ctypes.byref(p), ctypes.byref(n)))
    return int(p.value or 0), int(n.value)


def fill_uniform(T, d_out, count: int, seed: int, first_element: int = 0, stream=0) -> None:
    """Seeded U[-1,1) complex values (same formula as the test oracle's generator)."""
    _raise(lib().thff_fill_uniform(_precision(T), _ptr(d_out), int(count),
                                   int(seed) & (2**64 - 1), int(first_element), _stream(stream)))


def copy_nt(d_dst, d_src, nbytes: int, stream=0) -> None:
    """Non-temporal 16-byte streaming copy (the bandwidth ceiling bench.py reports)."""
    _raise(lib().thff_copy_nt(_ptr(d_dst), _ptr(d_src), int(nbytes), _stream(stream)))


def transforms_per_block(N: int) -> int:
    """Transforms per 256-lane workgroup of the global kernel."""
    return 256 * 16 // int(N)


def fft(x, forward: bool = True, out=None):
    """Transform the last axis of a CUDA tensor (complex64 or float16[..., N, 2]).

    A convenience over ThunderFFT_global.  ``out``, when given, must match
    ``x`` in dtype, shape and device, be contiguous and not overlap ``x``;
    every argument is checked (ValueError) before any HIP call.  The table for
    (T, N) is initialised on the tensor's device if needed, and the length
    that was current for T before the call is made current again afterwards
    (its table is kept, so that costs no allocation).
    """
    import torch

    if x.dtype == torch.complex64:
        T, n = "float", x.shape[-1]
    elif x.dtype == torch.float16 and x.dim() >= 2 and x.shape[-1] == 2:
        T, n = "half", x.shape[-2]
    else:
        raise ValueError("fft expects complex64 or float16[..., N, 2] tensors")
    if n not in SUPPORTED_N:
        raise ValueError(f"fft: unsupported FFT size {n} (supported: {SUPPORTED_N})")
    if out is not None:
        if out.dtype != x.dtype or tuple(out.shape) != tuple(x.shape) or out.device != x.device:
            raise ValueError("fft: out must match x in dtype, shape and device")
        if not out.is_contiguous():
            raise ValueError("fft: out must be contiguous")
        nbytes = x.numel() * x.element_size()
        if nbytes and (x.data_ptr() < out.data_ptr() + nbytes and
                       out.data_ptr() < x.data_ptr() + nbytes):
            raise ValueError("fft: out must not overlap x")
    if not x.is_cuda:
        raise ValueError("fft expects a device tensor (there is no CPU path)")
    x = x.contiguous()
    if out is None:
        out = torch.empty_like(x)
    batch = x.numel() // (n * (2 if T == "half" else 1))
    if batch == 0:
        return out
    with torch.cuda.device(x.device):
        previous = twiddle_info(T)[1]
        if previous != n:
            ThunderFFTInitialize(T, n)
        try:
            ThunderFFT_global(T, n, forward, x, out, batch, torch.cuda.current_stream(x.device))
        finally:
            if previous not in (0, n):
                ThunderFFTInitialize(T, previous)
    return out
