"""What the tensor functions hand to the kernels, on the CPU: the calls on device buffers are
replaced by ones that record their arguments."""
import contextlib

import pytest
import torch

import thunderfft_amd as thff
from thunderfft_amd import sequence

CALLS = ("ThunderFFT_gated_scan_async", "ThunderFFT_gated_scan_backward_async", "ThunderFFT_layer_norm_async",
         "ThunderFFT_layer_norm_backward_async")


@pytest.fixture
def calls(monkeypatch):
    """{name: (positional, by name)} of the last call of each kind; outputs stay as allocated."""
    made = {}

    def recorder(name):
        def call(*args, **named):
            made[name] = (args, named)
        return call

    for name in CALLS:
        monkeypatch.setattr(thff, name, recorder(name))
    monkeypatch.setattr(sequence, "_device_tensor", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: 0)
    return made


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=str)
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(before)


def floats(shape, **more):
    return torch.zeros(shape, dtype=torch.float32, **more)


@pytest.mark.parametrize("layout", ["channels_last", "channels_first"])
def test_scan_buffers_are_float_whatever_the_default(calls, default_dtype, layout):
    """The kernels write 4 bytes a state, also where torch's default type has 2 or 8."""
    dims = (2, 9, 6) if layout == "channels_last" else (2, 6, 9)
    x, gate, state = (floats(d, requires_grad=True) for d in (dims, dims, (2, 6)))
    y, last = thff.gated_scan(x, gate, state, layout=layout)
    torch.autograd.backward([y, last], [torch.zeros_like(y), torch.zeros_like(last)])
    _, forward = calls["ThunderFFT_gated_scan_async"]
    _, backward = calls["ThunderFFT_gated_scan_backward_async"]
    for t in (forward["d_state_out"], backward["d_dstate_out"], backward["d_dstate_in"]):
        assert t.dtype == torch.float32 and t.shape == (2, 6) and t.is_contiguous()
    assert last.dtype == torch.float32 and state.grad.dtype == torch.float32


def test_norm_buffers_are_float_whatever_the_default(calls, default_dtype):
    x, weight, bias = (floats(d, requires_grad=True) for d in ((5, 8), (8,), (8,)))
    y = thff.layer_norm(x, weight, bias)
    y.backward(torch.zeros_like(y))
    _, forward = calls["ThunderFFT_layer_norm_async"]
    args, _ = calls["ThunderFFT_layer_norm_backward_async"]
    for t, rows in ((forward["d_mean"], 5), (forward["d_rstd"], 5), (args[7], 8), (args[8], 8)):
        assert t.dtype == torch.float32 and t.shape == (rows,)
    assert weight.grad.dtype == torch.float32 and bias.grad.dtype == torch.float32
