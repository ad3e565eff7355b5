"""The sequence operators on torch tensors, with their gradients.

    y, state = gated_scan(x, gate, state=None, lengths=None, layout="channels_last")
    y = layer_norm(x, weight=None, bias=None, eps=1e-5)

Both run the HIP kernels on the current stream of the tensors' device and raise
ValueError for arguments that the kernels cannot take; there is no CPU path.  Buffers
come from torch's allocator, so that calls on several streams do not share any.
"""
from __future__ import annotations

import torch

import thunderfft_amd as thff

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _device_tensor(name, t, dtype=None, shape=None, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor (there is no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _rows(t):
    """(t, elements between its rows) if all rows of the last axis are equally far apart and
    do not overlap; else a contiguous copy."""
    *outer, last = t.shape
    if t.numel() == 0:
        return t, None
    stride = next((t.stride(i) for i in reversed(range(len(outer))) if outer[i] > 1), last)
    expected = stride
    fits = (last == 1 or t.stride(-1) == 1) and stride >= last
    for i in reversed(range(len(outer))):
        fits = fits and (outer[i] == 1 or t.stride(i) == expected)
        expected *= outer[i]
    if not fits:
        t, stride = t.contiguous(), last
    return t, stride


def _shape_of(x, x_stride, gate_stride, layout, y_stride=None):
    batch, n, channels = x.shape if layout == "channels_last" else (x.shape[0], x.shape[2], x.shape[1])
    return thff.ScanShape(x.dtype, batch, n, channels, layout=layout, x_stride=x_stride,
                          gate_stride=gate_stride, y_stride=y_stride)


def _bytes(count, device):
    return torch.empty(count, dtype=torch.uint8, device=device)


def _floats(*shape, device):
    """A buffer of states, statistics or weights' gradients: the kernels have them in float32,
    whatever torch's default type is."""
    return torch.empty(shape, dtype=torch.float32, device=device)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, lengths, layout):
        (x, x_stride), (gate, gate_stride) = _rows(x), _rows(gate)
        shape = _shape_of(x, x_stride, gate_stride, layout)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = _floats(shape.batch, shape.channels, device=x.device)
        train = any(ctx.needs_input_grad[:3])
        with torch.cuda.device(x.device):
            saved = _bytes(shape.saved_bytes(), x.device) if train else None
            thff.ThunderFFT_gated_scan_async(
                shape, x, gate, y, d_state_in=state, d_state_out=last, d_lengths=lengths,
                d_saved=saved, d_workspace=_bytes(shape.workspace_bytes(), x.device),
                stream=torch.cuda.current_stream())
        if train:
            ctx.save_for_backward(x, gate, lengths, saved)
            ctx.layout = layout
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, gate, lengths, saved = ctx.saved_tensors
        (dy, dy_stride), (x, x_stride), (gate, gate_stride) = _rows(dy), _rows(x), _rows(gate)
        # The kernels take one stride for x and its gradient, and one for the gate and its own.
        # Halves of a projection have theirs as halves of one buffer; rows that are further apart
        # otherwise are read from dense copies, so that the gradients need no such gaps.
        last = x.shape[-1]
        if x_stride == gate_stride == 2 * last:
            both = torch.empty(*x.shape[:-1], 2 * last, dtype=x.dtype, device=x.device)
            dx, dgate = both[..., :last], both[..., last:]
        else:
            x, gate, x_stride, gate_stride = x.contiguous(), gate.contiguous(), None, None
            dx, dgate = torch.empty_like(x), torch.empty_like(gate)
        shape = _shape_of(x, x_stride, gate_stride, ctx.layout, dy_stride)
        dstate = _floats(shape.batch, shape.channels, device=x.device)
        dlast = dlast.contiguous()
        with torch.cuda.device(x.device):
            thff.ThunderFFT_gated_scan_backward_async(
                shape, dy, x, gate, saved, dx, dgate, d_dstate_out=dlast, d_dstate_in=dstate,
                d_lengths=lengths, d_workspace=_bytes(shape.workspace_bytes(), x.device),
                stream=torch.cuda.current_stream())
        needs = ctx.needs_input_grad
        return (dx if needs[0] else None, dgate if needs[1] else None,
                dstate if needs[2] else None, None, None)


def gated_scan(x, gate, state=None, lengths=None, layout="channels_last"):
    """(y, last states) of h[t] = f[t] h[t-1] + (1 - f[t]) x[t], f = sigmoid(gate), y = h.

    x and gate: float32, float16 or bfloat16 of one shape, (batch, n, channels) or, with
    layout "channels_first", (batch, channels, n); halves of one projection are read in
    place, backward too, and have the halves of one buffer as gradients.  state: float32 (batch, channels) before the first step, None for zeros.
    lengths: int32 (batch,), steps from there on are left out and give y = 0.  The last
    states are float32 (batch, channels).  Differentiable (once) by x, gate and state.
    """
    if layout not in thff.ScanShape.LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(thff.ScanShape.LAYOUTS)} (got {layout!r})")
    _device_tensor("x", x)
    if x.dtype not in _TYPES or x.dim() != 3:
        raise ValueError("x must be float32, float16 or bfloat16 of three axes")
    _device_tensor("gate", gate, x.dtype, x.shape, x.device)
    channels = x.shape[2 if layout == "channels_last" else 1]
    if state is not None:
        _device_tensor("state", state, torch.float32, (x.shape[0], channels), x.device)
        state = state.contiguous()
    if lengths is not None:
        _device_tensor("lengths", lengths, torch.int32, (x.shape[0],), x.device)
        lengths = lengths.contiguous()
    return _GatedScan.apply(x, gate, state, lengths, layout)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, x_stride = _rows(x)
        cols = x.shape[-1]
        rows = x.numel() // cols
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        train = any(ctx.needs_input_grad[:3])
        mean = _floats(rows, device=x.device) if train else None
        rstd = _floats(rows, device=x.device) if train else None
        with torch.cuda.device(x.device):
            thff.ThunderFFT_layer_norm_async(x.dtype, x, weight, bias, eps, y, rows, cols,
                                             d_mean=mean, d_rstd=rstd, x_stride=x_stride,
                                             stream=torch.cuda.current_stream())
        if train:
            ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        needs = ctx.needs_input_grad
        (dy, dy_stride), (x, x_stride) = _rows(dy), _rows(x)
        cols = x.shape[-1]
        rows = x.numel() // cols
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dweight = _floats(cols, device=x.device) if needs[1] else None
        dbias = _floats(cols, device=x.device) if needs[2] else None
        with torch.cuda.device(x.device):
            workspace = (_bytes(thff.layer_norm_workspace_bytes(rows, cols), x.device)
                         if needs[1] or needs[2] else None)
            thff.ThunderFFT_layer_norm_backward_async(
                x.dtype, dy, x, mean, rstd, weight, dx, dweight, dbias, workspace, rows, cols,
                dy_stride=dy_stride, x_stride=x_stride, stream=torch.cuda.current_stream())
        return dx if needs[0] else None, dweight, dbias, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.

    x: float32, float16 or bfloat16 with at least one axis; weight and bias: float32
    (cols,), None for ones and zeros.  Differentiable (once) by x, weight and bias.
    """
    _device_tensor("x", x)
    if x.dtype not in _TYPES or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be float32, float16 or bfloat16 with a last axis of at least 1")
    if not eps >= 0:
        raise ValueError("eps must be nonnegative")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _device_tensor(name, t, torch.float32, x.shape[-1:], x.device)
    return _LayerNorm.apply(x, None if weight is None else weight.contiguous(),
                            None if bias is None else bias.contiguous(), float(eps))
