"""The operators of a state space block on torch tensors, with their gradients.

    y, state = short_conv(x, weight, bias=None, state=None, lengths=None, silu=True)
    y, state = state_scan(x, delta, a, b, c, skip=None, gate=None, delta_bias=None, state=None,
                          lengths=None)
    y = rms_norm(x, weight=None, eps=1e-5)
    y, sums = rms_norm(x, weight, residual, eps=1e-5)
    q, scales[, sums] = rms_norm_8bit(x, weight=None, residual=None, eps=1e-5, block=128)

All run the HIP kernels on the current stream of the tensors' device and raise ValueError for
arguments that the kernels cannot take; there is no CPU path.  Buffers come from torch's
allocator, so that calls on several streams do not share any.
"""
from __future__ import annotations

import torch

import thunderfft_amd as thff

from .sequence import _TYPES, _bytes, _device_tensor, _floats, _rows


def _values(name, t, axes):
    _device_tensor(name, t)
    if t.dtype not in _TYPES or t.dim() != axes:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 of {axes} axes")


def _optional(name, t, dtype, shape, device):
    """A contiguous argument of that type and shape, or None."""
    if t is None:
        return None
    _device_tensor(name, t, dtype, shape, device)
    return t.contiguous()


# Elements between rows that the scan takes at most.
_FARTHEST = 1 << 24


def _near_rows(t):
    """As _rows, with a dense copy of rows further apart than the scan takes (the last steps of long
    sequences, say)."""
    t, stride = _rows(t)
    return (t, stride) if stride is None or stride <= _FARTHEST else (t.contiguous(), t.shape[-1])


def _like(t, stride):
    """A gradient's buffer for rows `stride` apart (None: no rows): the same distance, as the kernels
    take one for both, without memory for what lies between the last row and the next."""
    last = t.shape[-1]
    if stride is None or stride == last:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    strides = [1]
    for size in reversed(t.shape[1:]):
        strides.insert(0, stride if len(strides) == 1 else strides[0] * size)
    return torch.empty_strided(t.shape, strides, dtype=t.dtype, device=t.device)


def _trained(*tensors):
    """Whether a backward pass may follow."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu):
        ctx.set_materialize_grads(False)
        x, x_stride = _rows(x)
        batch, n, channels = x.shape
        shape = thff.ConvShape(x.dtype, batch, n, channels, weight.shape[1], silu, x_stride)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = torch.empty(batch, weight.shape[1] - 1, channels, dtype=x.dtype, device=x.device)
        with torch.cuda.device(x.device):
            thff.ThunderFFT_short_conv_async(shape, x, weight, bias, y, d_state_in=state, d_state_out=last,
                                             d_lengths=lengths, stream=torch.cuda.current_stream())
        if any(ctx.needs_input_grad[:4]):
            ctx.save_for_backward(x, weight, bias, state, lengths)
            ctx.silu = silu
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy
        (dy, dy_stride), (x, x_stride) = _rows(dy), _rows(x)
        batch, n, channels = x.shape
        needs, width = ctx.needs_input_grad, weight.shape[1]
        shape = thff.ConvShape(x.dtype, batch, n, channels, width, ctx.silu, x_stride, dy_stride)
        dx = _like(x, x_stride)
        dweight = _floats(channels, width, device=x.device) if needs[1] else None
        dbias = _floats(channels, device=x.device) if needs[2] else None
        dstate = torch.empty(state.shape, dtype=x.dtype, device=x.device) if needs[3] else None
        dlast = None if dlast is None else dlast.contiguous()
        with torch.cuda.device(x.device):
            workspace = _bytes(shape.workspace_bytes(), x.device) if needs[1] or needs[2] else None
            thff.ThunderFFT_short_conv_backward_async(
                shape, dy, x, weight, bias, dx, dweight, dbias, d_state_in=state, d_dstate_out=dlast, d_dstate_in=dstate,
                d_lengths=lengths, d_workspace=workspace, stream=torch.cuda.current_stream())
        return dx if needs[0] else None, dweight, dbias, dstate, None, None


def short_conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    """(y, last state) of y[t] = silu(bias + sum_k weight[:, k] x[t - width + 1 + k]) in each channel.

    x: float32, float16 or bfloat16 (batch, n, channels), rows of a projection are read in place.
    weight: float32 (channels, width), width 2 to 4; bias: float32 (channels,), None for zeros.
    state: the width - 1 values before the first step, of x's type, (batch, width - 1, channels),
    None for zeros; the last state is those before the next one.  lengths: int32 (batch,), steps from
    there on are left out and give y = 0.  silu=False leaves the activation out.  Differentiable
    (once) by x, weight, bias and state.
    """
    _values("x", x, 3)
    batch, _, channels = x.shape
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        raise ValueError("weight must be of shape (channels, width), width 2 to 4")
    width = weight.shape[1]
    _device_tensor("weight", weight, torch.float32, (channels, width), x.device)
    return _ShortConv.apply(x, weight.contiguous(), _optional("bias", bias, torch.float32, (channels,), x.device),
                            _optional("state", state, x.dtype, (batch, width - 1, channels), x.device),
                            _optional("lengths", lengths, torch.int32, (batch,), x.device), bool(silu))


class _StateScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, a, b, c, skip, gate, delta_bias, state, lengths, train):
        ctx.set_materialize_grads(False)
        values = [x, delta, gate, b.flatten(2), c.flatten(2)]
        (x, xs), (delta, ds), gate_rows, (b_rows, bs), (c_rows, cs) = (
            _near_rows(t) if t is not None else (None, None) for t in values)
        batch, n, channels = x.shape
        order, groups = b.shape[3], b.shape[2]
        shape = thff.StateShape(x.dtype, batch, n, channels, order, groups, xs, ds, gate_rows[1], bs, cs)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = _floats(batch, channels, order, device=x.device)
        with torch.cuda.device(x.device):
            saved = _bytes(shape.saved_bytes(), x.device) if train else None
            thff.ThunderFFT_state_scan_async(
                shape, x, delta, a, b_rows, c_rows, y, d_skip=skip, d_gate=gate_rows[0], d_delta_bias=delta_bias,
                d_state_in=state, d_state_out=last, d_lengths=lengths, d_saved=saved,
                d_workspace=_bytes(shape.forward_bytes(), x.device), stream=torch.cuda.current_stream())
        if train:
            ctx.save_for_backward(x, delta, a, b_rows, c_rows, skip, gate_rows[0], delta_bias, lengths, saved)
            ctx.groups = groups
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, delta, a, b, c, skip, gate, delta_bias, lengths, saved = ctx.saved_tensors
        needs, device = ctx.needs_input_grad, x.device
        dy = torch.zeros_like(x) if dy is None else dy
        values = [dy, x, delta, gate, b, c]
        (dy, dys), (x, xs), (delta, ds), (gate, gs), (b, bs), (c, cs) = (
            _near_rows(t) if t is not None else (None, None) for t in values)
        batch, n, channels = x.shape
        order = a.shape[1]
        shape = thff.StateShape(x.dtype, batch, n, channels, order, ctx.groups, xs, ds, gs, bs, cs, dys)
        dx, ddelta, db, dc = _like(x, xs), _like(delta, ds), _like(b, bs), _like(c, cs)
        dgate = _like(gate, gs) if gate is not None else None
        da = _floats(channels, order, device=device)
        dskip = _floats(channels, device=device) if needs[5] else None
        dbias = _floats(channels, device=device) if needs[7] else None
        dstate = _floats(batch, channels, order, device=device) if needs[8] else None
        dlast = None if dlast is None else dlast.contiguous()
        with torch.cuda.device(device):
            thff.ThunderFFT_state_scan_backward_async(
                shape, dy, x, delta, a, b, c, saved, dx, ddelta, da, db, dc, d_skip=skip, d_dskip=dskip, d_gate=gate,
                d_dgate=dgate, d_delta_bias=delta_bias, d_ddelta_bias=dbias, d_dstate_out=dlast, d_dstate_in=dstate,
                d_lengths=lengths, d_workspace=_bytes(shape.workspace_bytes(), device),
                stream=torch.cuda.current_stream())
        shared = (batch, n, ctx.groups, order)
        got = (dx, ddelta, da, db.unflatten(2, shared[2:]), dc.unflatten(2, shared[2:]), dskip, dgate, dbias, dstate, None, None)
        return tuple(g if need else None for g, need in zip(got, needs))


def state_scan(x, delta, a, b, c, skip=None, gate=None, delta_bias=None, state=None, lengths=None):
    """(y, last states) of the state space scan: with dt = softplus(delta + delta_bias), for each
    channel and each of its states h[t] = exp(dt a) h[t-1] + dt x b, y = (sum of c h + skip x)
    silu(gate).

    x, delta and gate: float32, float16 or bfloat16 (batch, n, channels); without a gate y is the
    sum.  a: float32 (channels, order), order 1 to 64.  b and c: of x's type, (batch, n, order), or
    (batch, n, groups, order), where the channels fall into that many groups side by side.  Slices of
    a projection's rows are read in place (rows more than 2^24 elements apart are copied).  skip and delta_bias: float32 (channels,), None for zeros.
    state: float32 (batch, channels, order) before the first step, None for zeros; the last states
    are alike.  lengths: int32 (batch,), steps from there on are left out and give y = 0.
    Differentiable (once) by all but lengths.
    """
    _values("x", x, 3)
    batch, n, channels = x.shape
    if not isinstance(a, torch.Tensor) or a.dim() != 2 or not 1 <= a.shape[1] <= 64:
        raise ValueError("a must be of shape (channels, order), order 1 to 64")
    order = a.shape[1]
    for name, t in (("b", b), ("c", c)):
        if not isinstance(t, torch.Tensor) or t.dim() not in (3, 4):
            raise ValueError(f"{name} must be of shape (batch, n, order) or (batch, n, groups, order)")
    b, c = (t.unsqueeze(2) if t.dim() == 3 else t for t in (b, c))
    groups = b.shape[2]
    if groups < 1 or channels % groups != 0:
        raise ValueError(f"groups must divide the channels (got {groups} groups, {channels} channels)")
    _device_tensor("delta", delta, x.dtype, x.shape, x.device)
    _device_tensor("a", a, torch.float32, (channels, order), x.device)
    _device_tensor("b", b, x.dtype, (batch, n, groups, order), x.device)
    _device_tensor("c", c, x.dtype, (batch, n, groups, order), x.device)
    if gate is not None:
        _device_tensor("gate", gate, x.dtype, x.shape, x.device)
    skip, delta_bias = (_optional(name, t, torch.float32, (channels,), x.device)
                        for name, t in (("skip", skip), ("delta_bias", delta_bias)))
    state = _optional("state", state, torch.float32, (batch, channels, order), x.device)
    lengths = _optional("lengths", lengths, torch.int32, (batch,), x.device)
    train = _trained(x, delta, a, b, c, skip, gate, delta_bias, state)
    return _StateScan.apply(x, delta, a.contiguous(), b, c, skip, gate, delta_bias, state, lengths, train)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, train):
        ctx.set_materialize_grads(False)
        (x, x_stride), (residual, residual_stride) = _rows(x), _rows(residual) if residual is not None else (None, None)
        cols = x.shape[-1]
        rows = x.numel() // cols
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
        rstd = _floats(rows, device=x.device) if train else None
        with torch.cuda.device(x.device):
            thff.ThunderFFT_rms_norm_async(x.dtype, x, weight, eps, y, rows, cols, d_residual=residual, d_sum=total,
                                           d_rstd=rstd, x_stride=x_stride, residual_stride=residual_stride,
                                           stream=torch.cuda.current_stream())
        if train:
            # The sums are an output: a later change in place is noticed.
            ctx.save_for_backward(x if total is None else total, weight, rstd)
        return (y, total) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        total, weight, rstd = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dy = torch.zeros_like(total) if dy is None else dy
        (dy, dy_stride), (total, sum_stride) = _rows(dy), _rows(total)
        dsum, dsum_stride = _rows(dsum) if dsum is not None else (None, None)
        cols = total.shape[-1]
        rows = total.numel() // cols
        dx = torch.empty(total.shape, dtype=total.dtype, device=total.device)
        dweight = _floats(cols, device=total.device) if needs[1] else None
        with torch.cuda.device(total.device):
            workspace = _bytes(thff.rms_norm_workspace_bytes(rows, cols), total.device) if needs[1] else None
            thff.ThunderFFT_rms_norm_backward_async(
                total.dtype, dy, total, rstd, weight, dx, dweight, workspace, rows, cols, d_dsum=dsum, dy_stride=dy_stride,
                sum_stride=sum_stride, dsum_stride=dsum_stride, stream=torch.cuda.current_stream())
        return dx if needs[0] else None, dweight, dx if needs[2] else None, None, None


def _norm_arguments(x, weight, residual, eps):
    _device_tensor("x", x)
    if x.dtype not in _TYPES or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be float32, float16 or bfloat16 with a last axis of at least 1")
    if not eps >= 0:
        raise ValueError("eps must be nonnegative")
    if residual is not None:
        _device_tensor("residual", residual, x.dtype, x.shape, x.device)
    return _optional("weight", weight, torch.float32, x.shape[-1:], x.device)


def rms_norm(x, weight=None, residual=None, eps=1e-5):
    """s / sqrt(mean(s^2) + eps) * weight over the last axis, with s = x; with a residual
    s = x + residual, rounded to x's type, and the result is (y, s).

    x and residual: float32, float16 or bfloat16 of one shape; weight: float32 (cols,), None for
    ones.  Differentiable (once) by x, weight and residual.
    """
    weight = _norm_arguments(x, weight, residual, eps)
    return _RmsNorm.apply(x, weight, residual, float(eps), _trained(x, weight, residual))


@torch.no_grad()
def rms_norm_8bit(x, weight=None, residual=None, eps=1e-5, block=128):
    """(q, scales) with y of rms_norm near q * scales: q is torch.float8_e4m3fn of x's shape, scales
    float32 with one for every `block` columns (128, or None for one a row) in the last axis's place,
    the largest |y| of them / 448.  With a residual (q, scales, x + residual).  Not differentiable.
    """
    weight = _norm_arguments(x, weight, residual, eps)
    if block not in (128, None):
        raise ValueError("block must be 128 or None")
    cols = x.shape[-1]
    block = cols if block is None else block
    (x, x_stride), (residual, residual_stride) = _rows(x), _rows(residual) if residual is not None else (None, None)
    rows = x.numel() // cols
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = _floats(*x.shape[:-1], -(-cols // block), device=x.device)
    total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    with torch.cuda.device(x.device):
        thff.ThunderFFT_rms_norm_8bit_async(x.dtype, x, weight, float(eps), q, scales, rows, cols, block,
                                            d_residual=residual, d_sum=total, x_stride=x_stride,
                                            residual_stride=residual_stride, stream=torch.cuda.current_stream())
    return (q, scales) if residual is None else (q, scales, total)
