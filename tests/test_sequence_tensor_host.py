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


def halves(both):
    last = both.shape[-1] // 2
    return both[..., :last], both[..., last:]


# x and the gate as programs have them, and whether their gradients' rows lie as theirs do.
PLACES = {
    "halves": (lambda: halves(torch.zeros(2, 9, 12)), True),
    "swapped halves": (lambda: halves(torch.zeros(2, 9, 12))[::-1], True),
    "halves of two": (lambda: (halves(torch.zeros(2, 9, 12))[0], halves(torch.zeros(2, 9, 12))[1]), True),
    "halves of one step": (lambda: halves(torch.zeros(5, 1, 12)), True),
    "dense": (lambda: (torch.zeros(2, 9, 6), torch.zeros(2, 9, 6)), True),
    "one a half": (lambda: (halves(torch.zeros(2, 9, 12))[0], torch.zeros(2, 9, 6)), False),
    "thirds": (lambda: torch.zeros(2, 9, 18).chunk(3, -1)[:2], False),
    "transposed": (lambda: (torch.zeros(2, 6, 9).transpose(1, 2), torch.zeros(2, 6, 9).transpose(1, 2)), False),
    "expanded": (lambda: (torch.zeros(2, 1, 6).expand(2, 9, 6), torch.zeros(2, 9, 6)), False),
}


@pytest.mark.parametrize("layout", ["channels_last", "channels_first"])
@pytest.mark.parametrize("place", PLACES)
def test_backward_reads_in_place(calls, place, layout):
    """The backward call has the tensors that the forward call had, their rows as far apart as it is
    told, and gradients with the same; halves of a projection are not copied."""
    make, in_place = PLACES[place]
    x, gate = (v.detach().requires_grad_() for v in make())
    y, last = thff.gated_scan(x, gate, layout=layout)
    torch.autograd.backward([y, last], [torch.zeros_like(y), torch.zeros_like(last)])
    (ahead, fx, fgate, _), _ = calls["ThunderFFT_gated_scan_async"]
    (shape, _, bx, bgate, _, dx, dgate), _ = calls["ThunderFFT_gated_scan_backward_async"]

    def apart(t):
        return t.stride(1) if t.shape[1] > 1 else t.stride(0)

    for s, tensors in ((ahead, (fx, fgate)), (shape, (bx, bgate)), (shape, (dx, dgate))):
        for t, stride in zip(tensors, (s.x_stride, s.gate_stride)):
            assert t.shape == x.shape and t.stride(2) == 1 and apart(t) == (stride or t.shape[2])
            assert t.shape[1] == 1 or t.stride(0) == t.shape[1] * t.stride(1)
    assert dx.dtype == x.dtype and x.grad.shape == x.shape and gate.grad.shape == x.shape
    if in_place:
        assert bx.data_ptr() == x.data_ptr() and bgate.data_ptr() == gate.data_ptr()
