"""The sequence operators' refusals and sizes, all decided before any HIP call, and their
oracle against difference quotients, on the CPU."""
import ctypes

import pytest
import torch

import sequence_oracle as oracle
import thunderfft_amd as thff

A, B, C, D, E = 1 << 16, 2 << 16, 3 << 16, 4 << 16, 5 << 16  # never dereferenced


def shape(T="half", batch=2, n=300, channels=70, **more):
    return thff.ScanShape(T, batch, n, channels, **more)


def test_shapes_refused():
    for bad in (dict(batch=-1), dict(n=-1), dict(channels=-1)):
        with pytest.raises(ValueError, match="nonnegative"):
            shape(**bad).saved_bytes()
    for bad in (dict(batch=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(channels=(1 << 30) + 1)):
        with pytest.raises(ValueError, match="at most 2\\^30"):
            shape(**bad).workspace_bytes()
    with pytest.raises(ValueError, match="exceeds one launch"):
        shape(batch=1 << 16, channels=1 << 15).saved_bytes()
    for bad in (dict(x_stride=69), dict(gate_stride=69), dict(y_stride=-70)):
        with pytest.raises(ValueError, match="stride"):
            shape(**bad).saved_bytes()
    with pytest.raises(ValueError, match="stride"):
        shape(layout="channels_first", x_stride=299).saved_bytes()
    with pytest.raises(ValueError, match="stride"):
        shape(batch=1 << 30, n=1 << 30, channels=1, x_stride=1 << 30).saved_bytes()
    with pytest.raises(ValueError, match="layout"):
        shape(layout="channels_middle")
    with pytest.raises(ValueError, match="float, half and bfloat16"):
        shape(T="double")
    with pytest.raises(ValueError, match="out of range"):
        shape(batch=1 << 31)
    for field, value in (("precision", 3), ("layout", 2)):
        s = shape()
        setattr(s, field, value)
        with pytest.raises(ValueError):
            s.saved_bytes()
    L = thff.lib()
    assert L.thff_gated_scan(None, A, B, C, 0, 0, 0, 0, 0, 0, 0) == thff.THFF_EINVAL
    assert L.thff_gated_scan_saved_bytes(None) == thff.THFF_EINVAL


def test_launch_limits():
    """Shapes whose workgroups one launch does not have are refused; the largest ones are not."""
    for layout in ("channels_last", "channels_first"):
        with pytest.raises(ValueError, match="exceeds one launch"):
            shape(batch=1 << 20, n=1 << 28, channels=64, layout=layout).saved_bytes()
        assert shape(batch=1 << 30, n=2, channels=1, layout=layout).saved_bytes() > 0
        assert shape(batch=1 << 20, n=3, channels=64, layout=layout).saved_bytes() > 0
        assert shape(batch=1, n=1 << 30, channels=128, layout=layout).workspace_bytes() > 0


def test_sizes():
    """Sizes are counted, not negative, and grow with what has to be kept."""
    for layout in ("channels_last", "channels_first"):
        s = [shape(n=n, layout=layout).saved_bytes() for n in (0, 1, 300, 3000, 1 << 30)]
        assert s[0] >= 0 and s == sorted(s)
        assert all(shape(n=n, layout=layout).workspace_bytes() >= 0 for n in (0, 1, 300, 3000, 1 << 30))
    assert thff.layer_norm_workspace_bytes(0, 1) >= 0
    assert thff.layer_norm_workspace_bytes(1 << 40, 1 << 20) >= 0


@pytest.mark.parametrize("call", [thff.ThunderFFT_gated_scan, thff.ThunderFFT_gated_scan_async])
def test_scan_refused(call):
    s = shape()
    w = dict(d_workspace=E)
    for x, gate, y in ((0, B, C), (A, 0, C), (A, B, 0)):
        with pytest.raises(ValueError, match="non-null"):
            call(s, x, gate, y, **w)
    for y in (A, B):
        with pytest.raises(ValueError, match="alias"):
            call(s, A, B, y, **w)
    for x, gate, y in ((A + 1, B, C), (A, B + 1, C), (A, B, C + 1)):
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, x, gate, y, **w)
    with pytest.raises(ValueError, match="element-aligned"):
        call(shape("float"), A + 2, B, C, **w)
    for bad in ("d_state_in", "d_state_out", "d_slots", "d_lengths"):
        with pytest.raises(ValueError, match="4-byte aligned"):
            call(s, A, B, C, **{bad: D + 2}, **w)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(s, A, B, C, d_saved=D + 8, **w)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(s, A, B, C, d_workspace=D + 8)
    with pytest.raises(ValueError, match="states"):
        call(shape(states=-1), A, B, C, d_slots=D, **w)
    with pytest.raises(ValueError, match="nonnegative"):
        call(shape(n=-1), A, B, C)
    # A shape with nothing to do is done, whatever the pointers.
    call(shape(batch=0), 0, 0, 0)
    call(shape(channels=0), 0, 0, 0)
    with pytest.raises(TypeError):
        call(s, "x", B, C)


@pytest.mark.parametrize("call", [thff.ThunderFFT_gated_scan_backward,
                                  thff.ThunderFFT_gated_scan_backward_async])
def test_scan_backward_refused(call):
    s = shape()
    good = [A, B, C, D, E, 6 << 16]  # dy, x, gate, saved, dx, dgate
    w = dict(d_workspace=7 << 16)
    for k in (0, 1, 2, 4, 5):
        args = list(good)
        args[k] = 0
        with pytest.raises(ValueError, match="non-null"):
            call(s, *args, **w)
        args[k] = good[k] + 1
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, *args, **w)
    for out in (4, 5):
        for k in {0, 1, 2, 4, 5} - {out}:
            args = list(good)
            args[out] = args[k]
            with pytest.raises(ValueError, match="alias"):
                call(s, *args, **w)
    for bad in ("d_dstate_out", "d_dstate_in", "d_lengths"):
        with pytest.raises(ValueError, match="4-byte aligned"):
            call(s, *good, **{bad: (8 << 16) + 2}, **w)
    args = list(good)
    args[3] += 4
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(s, *args, **w)
    args[3] = 0
    if s.saved_bytes():
        with pytest.raises(ValueError, match="saved"):
            call(s, *args, **w)
    call(shape(batch=0), 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("twin", ["", "_async"])
def test_norm_refused(twin):
    forward = getattr(thff, "ThunderFFT_layer_norm" + twin)
    backward = getattr(thff, "ThunderFFT_layer_norm_backward" + twin)
    with pytest.raises(ValueError, match="float, half and bfloat16"):
        forward("double", A, B, C, 1e-5, D, 4, 8)
    for rows, cols, what in ((-1, 8, "rows"), (4, 0, "cols"), (4, -8, "cols"), (4, (1 << 30) + 1, "cols"),
                             (4, 1 << 32, "out of range")):
        with pytest.raises(ValueError, match=what):
            forward("half", A, B, C, 1e-5, D, rows, cols)
        with pytest.raises(ValueError, match=what):
            backward("half", A, B, C, D, E, 6 << 16, 0, 0, 0, rows, cols)
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            forward("half", A, B, C, eps, D, 4, 8)
    for x, y, what in ((0, D, "non-null"), (A, 0, "non-null"), (A, A, "alias"), (A + 1, D, "element"),
                       (A, D + 1, "element")):
        with pytest.raises(ValueError, match=what):
            forward("half", x, B, C, 1e-5, y, 4, 8)
    for k in range(4):
        extra = [B, C, 0, 0]
        extra[k] = E + 2
        with pytest.raises(ValueError, match="4-byte"):
            forward("half", A, extra[0], extra[1], 1e-5, D, 4, 8, d_mean=extra[2], d_rstd=extra[3])
    for more in (dict(x_stride=7), dict(y_stride=7), dict(x_stride=-8)):
        with pytest.raises(ValueError, match="stride"):
            forward("half", A, B, C, 1e-5, D, 4, 8, **more)
    forward("half", 0, 0, 0, 1e-5, 0, 0, 8)  # no rows

    good = [A, B, C, D, 0, E]  # dy, x, mean, rstd, weight, dx
    for k in (0, 1, 2, 3, 5):
        args = list(good)
        args[k] = 0
        with pytest.raises(ValueError, match="non-null"):
            backward("half", *args, 0, 0, 0, 4, 8)
    for k, step, what in ((0, 1, "element"), (1, 1, "element"), (5, 1, "element"), (2, 2, "4-byte"), (3, 2, "4-byte")):
        args = list(good)
        args[k] += step
        with pytest.raises(ValueError, match=what):
            backward("half", *args, 0, 0, 0, 4, 8)
    for k in (0, 1):
        args = list(good)
        args[5] = args[k]
        with pytest.raises(ValueError, match="alias"):
            backward("half", *args, 0, 0, 0, 4, 8)
    with pytest.raises(ValueError, match="dweight must not alias"):
        backward("half", *good, 7 << 16, 7 << 16, 8 << 16, 4, 8)
    with pytest.raises(ValueError, match="16-byte"):
        backward("half", *good, 7 << 16, 9 << 16, (8 << 16) + 4, 4, 8)
    for more in (dict(dy_stride=7), dict(x_stride=7), dict(dx_stride=7)):
        with pytest.raises(ValueError, match="stride"):
            backward("half", *good, 0, 0, 0, 4, 8, **more)
    backward("half", 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 8)  # no rows and no weights


def test_tensor_functions_refuse():
    """gated_scan and layer_norm have no CPU path and say so."""
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="device tensor"):
        thff.gated_scan(x, x)
    with pytest.raises(ValueError, match="layout"):
        thff.gated_scan(x, x, layout="time_first")
    with pytest.raises(ValueError, match="device tensor"):
        thff.layer_norm(x)


def test_c_struct_matches():
    """ScanShape has the C struct's fields, in its order and its size (no gaps)."""
    assert ctypes.sizeof(thff.ScanShape) == 6 * 4 + 3 * 8
    import os
    import re

    text = open(os.path.join(os.path.dirname(thff.LIB_PATH), "..", "include", "thunderfft", "thunderfft.h")).read()
    body = re.search(r"typedef struct thff_scan_shape \{(.*?)\}", text, re.S).group(1)
    names = re.findall(r"(\w+)\s*[,;]", body)
    assert names == [f[0] for f in thff.ScanShape._fields_]


@pytest.mark.parametrize("layout", ["channels_last", "channels_first"])
def test_scan_oracle_gradients(layout):
    """The oracle's gradients against central differences of its own values, in 64 bits:
    a step of 2^-17 leaves a truncation of 2^-34 of the third derivatives and a rounding
    of 2^-53 / 2^-17 of the sums, both far below 1e-7 of sums of order ten."""
    gen = torch.Generator().manual_seed(5)
    shape_ = (2, 9, 3) if layout == "channels_last" else (2, 3, 9)

    def normal(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    x, gate, state, dy, dstate = normal(*shape_), normal(*shape_), normal(2, 3), normal(*shape_), normal(2, 3)
    lengths = torch.tensor([9, 4])
    got = oracle.scan("float", layout, x, gate, state, lengths, dy, dstate)

    def loss(x, gate, state):
        v = oracle.scan("float", layout, x, gate, state, lengths)
        return float((v["y"][0] * dy).sum() + (v["state"][0] * dstate).sum())

    eps = 2.0 ** -17
    for name, at in (("dx", 0), ("dgate", 1), ("dstate", 2)):
        ins = [x, gate, state]
        v = normal(*ins[at].shape)
        up, down = list(ins), list(ins)
        up[at], down[at] = ins[at] + eps * v, ins[at] - eps * v
        along = float((got[name][0] * v).sum())
        assert abs((loss(*up) - loss(*down)) / (2 * eps) - along) < 1e-7, name


def test_norm_oracle_gradients():
    """As above, for layer norm."""
    gen = torch.Generator().manual_seed(6)

    def normal(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    x, w, b, dy = normal(4, 7), normal(7), normal(7), normal(4, 7)
    got = oracle.norm("float", x, w, b, 1e-5, dy)

    def loss(x, w, b):
        return float((oracle.norm("float", x, w, b, 1e-5)["y"][0] * dy).sum())

    eps = 2.0 ** -17
    for name, at in (("dx", 0), ("dweight", 1), ("dbias", 2)):
        ins = [x, w, b]
        v = normal(*ins[at].shape)
        up, down = list(ins), list(ins)
        up[at], down[at] = ins[at] + eps * v, ins[at] - eps * v
        along = float((got[name][0] * v).sum())
        assert abs((loss(*up) - loss(*down)) / (2 * eps) - along) < 1e-7, name


def test_norm_workspace_is_what_a_call_uses():
    """Partial sums of at most 256 workgroups, and none for rows that are not held in registers."""
    assert thff.layer_norm_workspace_bytes(300, 16384) == 8 * 256 * 16384
    assert thff.layer_norm_workspace_bytes(3, 16384) == 8 * 3 * 16384
    for rows, cols in ((3, 16385), (256, 65536), (256, 1 << 20), (1 << 40, 1 << 30)):
        assert thff.layer_norm_workspace_bytes(rows, cols) == 0
