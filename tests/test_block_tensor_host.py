"""What a state space block's tensor functions hand to the kernels, on the CPU: the calls on device
buffers are replaced by ones that record their arguments."""
import contextlib

import pytest
import torch

import thunderfft_amd as thff
from thunderfft_amd import block

CALLS = ("short_conv", "short_conv_backward", "state_scan", "state_scan_backward", "rms_norm", "rms_norm_8bit", "rms_norm_backward")


@pytest.fixture
def calls(monkeypatch):
    """{name: (positional, by name)} of the last call of each kind; outputs stay as allocated."""
    made = {}

    def recorder(name):
        def call(*args, **named):
            made[name] = (args, named)
        return call

    for name in CALLS:
        monkeypatch.setattr(thff, f"ThunderFFT_{name}_async", recorder(name))
    monkeypatch.setattr(block, "_device_tensor", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: 0)
    return made


@pytest.fixture(params=[torch.bfloat16, torch.float64], ids=str)
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(before)


def leaf(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, requires_grad=True)


def test_buffers_have_their_types_whatever_the_default(calls, default_dtype):
    """The kernels write float32 weights' gradients, states and statistics, and the convolution's states in
    the values' type, also where torch's default type is another."""
    half = torch.float16
    x, w, bias, state = leaf(2, 9, 6, dtype=half), leaf(6, 4), leaf(6), leaf(2, 3, 6, dtype=half)
    y, last = thff.short_conv(x, w, bias, state)
    torch.autograd.backward([y, last], [torch.zeros_like(y), torch.zeros_like(last)])
    args, named = calls["short_conv_backward"]
    assert args[5].dtype == half and args[6].dtype == args[7].dtype == torch.float32
    assert named["d_dstate_in"].dtype == named["d_dstate_out"].dtype == half and last.dtype == half

    delta, a, b, c, skip, gate, dbias, first = (leaf(2, 9, 6, dtype=half), leaf(6, 5), leaf(2, 9, 5, dtype=half),
                                                leaf(2, 9, 5, dtype=half), leaf(6), leaf(2, 9, 6, dtype=half), leaf(6), leaf(2, 6, 5))
    y, last = thff.state_scan(x, delta, a, b, c, skip, gate, dbias, first)
    torch.autograd.backward([y, last], [torch.zeros_like(y), torch.zeros_like(last)])
    args, named = calls["state_scan_backward"]
    dx, ddelta, da, db, dc = args[8:13]
    assert all(t.dtype == half for t in (dx, ddelta, db, dc, named["d_dgate"]))
    assert all(t.dtype == torch.float32 for t in (da, named["d_dskip"], named["d_ddelta_bias"], named["d_dstate_in"], last))
    assert b.grad.shape == b.shape and c.grad.shape == c.shape

    rows, weight, residual = leaf(5, 8, dtype=half), leaf(8), leaf(5, 8, dtype=half)
    y, total = thff.rms_norm(rows, weight, residual)
    torch.autograd.backward([y, total], [torch.zeros_like(y), torch.zeros_like(y)])
    args, named = calls["rms_norm_backward"]
    assert args[3].dtype == args[6].dtype == torch.float32 and args[5].dtype == half
    q, scales = thff.rms_norm_8bit(rows, weight, block=None)
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32 and scales.shape == (5, 1)


def test_slices_of_projections_are_read_in_place(calls):
    """Rows further apart than they are long: their distance is the shape's stride, for the gradients too."""
    rows = torch.zeros(2, 9, 40)
    x, gate, b, c = rows[..., :6], rows[..., 6:12], rows[..., 12:17], rows[..., 17:22]
    x, gate, b, c = (v.detach().requires_grad_() for v in (x, gate, b, c))
    delta, a = leaf(2, 9, 6), leaf(6, 5)
    y, _ = thff.state_scan(x, delta, a, b, c, gate=gate)
    y.sum().backward()
    for name in ("state_scan", "state_scan_backward"):
        args, named = calls[name]
        shape = args[0]
        assert [getattr(shape, k + "_stride") for k in ("x", "gate", "b", "c")] == [40] * 4 and shape.delta_stride == 6
        first = 1 if name == "state_scan" else 2
        assert args[first].data_ptr() == x.data_ptr() and named["d_gate"].data_ptr() == gate.data_ptr()
    args, named = calls["state_scan_backward"]
    for t in (args[8], args[11], args[12], named["d_dgate"]):
        assert t.stride(1) == 40 and t.stride(0) == 360 and t.stride(2) == 1
    y, _ = thff.short_conv(x, leaf(6, 3))
    y.sum().backward()
    args, _ = calls["short_conv_backward"]
    assert args[0].x_stride == 40 and args[5].stride() == (360, 40, 1)


def test_orders_that_rows_cannot_have_are_copied(calls):
    """Channels before steps, and one row for all: dense copies."""
    x = torch.zeros(2, 6, 9).transpose(1, 2)
    thff.short_conv(x, torch.zeros(6, 2))
    (shape, given, *_), _ = calls["short_conv"]
    assert given.is_contiguous() and shape.x_stride in (0, 6)
    thff.state_scan(x, x, torch.zeros(6, 3), torch.zeros(2, 1, 3).expand(2, 9, 3), torch.zeros(2, 9, 3))
    (shape, *arrays), _ = calls["state_scan"]
    assert all(arrays[k].is_contiguous() for k in (0, 1, 3, 4)) and shape.b_stride in (0, 3)
    thff.rms_norm(torch.zeros(3, 4, 5).transpose(0, 2))
    (_, given, *_), named = calls["rms_norm"]
    assert given.is_contiguous()


def test_nothing_is_kept_without_gradients(calls):
    with torch.no_grad():
        thff.state_scan(leaf(1, 2, 3), leaf(1, 2, 3), leaf(3, 4), leaf(1, 2, 4), leaf(1, 2, 4))
        thff.rms_norm(leaf(2, 3))
    assert calls["state_scan"][1]["d_saved"] is None and calls["rms_norm"][1]["d_rstd"] is None


def test_gradients_of_one_output(calls):
    """Outputs that nothing was made of give no gradients: dy is zeros, the states' and the sums' are left out."""
    x, w = leaf(2, 9, 6), leaf(6, 4)
    _, last = thff.short_conv(x, w)
    last.sum().backward()
    args, named = calls["short_conv_backward"]
    assert (args[1] == 0).all() and named["d_dstate_out"] is not None and named["d_dstate_in"] is None
    y, _ = thff.state_scan(x, leaf(2, 9, 6), leaf(6, 5), leaf(2, 9, 5), leaf(2, 9, 5))
    y.sum().backward()
    args, named = calls["state_scan_backward"]
    assert named["d_dstate_out"] is None and named["d_dskip"] is None and named["d_dgate"] is None
    rows = leaf(4, 5)
    y, _ = thff.rms_norm(rows, None, leaf(4, 5))
    y.sum().backward()
    args, named = calls["rms_norm_backward"]
    assert named["d_dsum"] is None and args[6] is None and args[7] is None


def test_rows_too_far_apart_for_the_scan_are_copied(calls):
    """The last steps of long sequences: rows more than 2^24 elements apart, which the kernels refuse, forward and
    as the gradient that comes back."""
    far = (1 << 25, 6, 1)
    x, delta, gate = (torch.empty_strided((2, 1, 6), far).requires_grad_() for _ in range(3))
    b, c = (torch.empty_strided((2, 1, 1, 5), (1 << 25, 6, 6, 1)).requires_grad_() for _ in range(2))
    y, last = thff.state_scan(x, delta, leaf(6, 5), b, c, gate=gate)
    (shape, *args), named = calls["state_scan"]
    assert [shape.x_stride, shape.delta_stride, shape.gate_stride, shape.b_stride, shape.c_stride] == [6, 6, 6, 5, 5]
    assert args[0].is_contiguous() and named["d_gate"].is_contiguous() and args[3].is_contiguous()
    y.backward(torch.empty_strided((2, 1, 6), far))
    (shape, *args), named = calls["state_scan_backward"]
    assert [shape.x_stride, shape.delta_stride, shape.gate_stride, shape.b_stride, shape.c_stride, shape.y_stride] == [6, 6, 6, 5, 5, 6]
    assert args[0].is_contiguous() and args[7].is_contiguous() and args[10].is_contiguous()
    assert all(t.grad.shape == t.shape for t in (x, delta, gate, b, c))
    # Rows as far apart as the kernels take are read in place.
    near = torch.empty_strided((2, 1, 6), (1 << 24, 6, 1))
    thff.state_scan(near, near, leaf(6, 5).detach(), near[..., :5], near[..., 1:])
    assert calls["state_scan"][0][0].x_stride == calls["state_scan"][0][0].b_stride == 1 << 24
