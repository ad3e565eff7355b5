"""A state space block's operators: refusals and sizes, all decided before any HIP call, and their
oracle against difference quotients, on the CPU."""
import ctypes
import os
import re

import pytest
import torch

import block_oracle as oracle
import thunderfft_amd as thff

A, B, C, D, E, F, G, H = (k << 16 for k in range(1, 9))  # never dereferenced


def conv_shape(T="half", batch=2, n=300, channels=70, width=4, **more):
    return thff.ConvShape(T, batch, n, channels, width, **more)


def state_shape(T="half", batch=2, n=300, channels=70, order=16, **more):
    return thff.StateShape(T, batch, n, channels, order, **more)


@pytest.mark.parametrize("make", [conv_shape, state_shape])
def test_shapes_refused(make):
    for bad in (dict(batch=-1), dict(n=-1), dict(channels=-1)):
        with pytest.raises(ValueError, match="nonnegative"):
            make(**bad).workspace_bytes()
    for bad in (dict(batch=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(channels=(1 << 30) + 1)):
        with pytest.raises(ValueError, match="at most 2\\^30"):
            make(**bad).workspace_bytes()
    with pytest.raises(ValueError, match="at most 2\\^31 - 256"):
        make(batch=1 << 16, channels=1 << 15).workspace_bytes()
    for bad in (dict(x_stride=69), dict(y_stride=-70), dict(batch=1 << 30, n=1 << 30, channels=1, x_stride=1 << 30)):
        with pytest.raises(ValueError, match="stride|one launch"):
            make(**bad).workspace_bytes()
    with pytest.raises(ValueError, match="float, half and bfloat16"):
        make(T="double")
    with pytest.raises(ValueError, match="out of range"):
        make(batch=1 << 31)
    s = make()
    s.precision = 3
    with pytest.raises(ValueError, match="float, half and bfloat16"):
        s.workspace_bytes()


def test_conv_shapes_refused():
    for width in (-1, 0, 1, 5):
        with pytest.raises(ValueError, match="width must be 2 to 4"):
            conv_shape(width=width).workspace_bytes()
    s = conv_shape()
    s.silu = 2
    with pytest.raises(ValueError, match="silu"):
        s.workspace_bytes()
    assert thff.lib().thff_short_conv_workspace_bytes(None) == thff.THFF_EINVAL
    assert thff.lib().thff_short_conv(None, A, B, 0, C, 0, 0, 0, 0, 0) == thff.THFF_EINVAL


def test_state_shapes_refused():
    for order in (-1, 0, 65):
        with pytest.raises(ValueError, match="order must be 1 to 64"):
            state_shape(order=order).saved_bytes()
    for groups in (-1, 0, 3, 71):
        with pytest.raises(ValueError, match="groups must divide"):
            state_shape(groups=groups).saved_bytes()
    for bad in (dict(delta_stride=69), dict(gate_stride=69), dict(b_stride=15), dict(c_stride=15),
                dict(groups=2, b_stride=31)):
        with pytest.raises(ValueError, match="stride"):
            state_shape(**bad).saved_bytes()
    for bad in ("x", "delta", "gate", "b", "c", "y"):
        with pytest.raises(ValueError, match="at most 2\\^24"):
            state_shape(**{bad + "_stride": (1 << 24) + 1}).saved_bytes()
        assert state_shape(**{bad + "_stride": 1 << 24}).saved_bytes() > 0
    with pytest.raises(ValueError, match="exceeds one launch"):
        state_shape(batch=1 << 28, n=1 << 30, channels=1, order=4).saved_bytes()
    assert thff.lib().thff_state_scan_saved_bytes(None) == thff.THFF_EINVAL
    assert thff.lib().thff_state_scan_workspace_bytes(None) == thff.THFF_EINVAL


def test_sizes():
    """Sizes are counted, not negative, and grow with what has to be kept."""
    for order in (1, 4, 5, 16, 17, 64):
        s = [state_shape(n=n, order=order).saved_bytes() for n in (0, 1, 300, 3000, 1 << 30)]
        assert s[0] == 0 and s == sorted(s)
        assert all(state_shape(n=n, order=order).workspace_bytes() > 0 for n in (0, 1, 300, 1 << 20))
        assert state_shape(n=1, order=order).forward_bytes() == 0 and state_shape(n=1 << 16, order=order).forward_bytes() > 0
    # Many channels leave no segments, and a forward call no scratch.
    assert state_shape(batch=8, n=4096, channels=2048).forward_bytes() == 0
    assert state_shape(channels=0).workspace_bytes() == 0
    # Past 32 bits: 2^30 sequences of a step.
    assert state_shape(batch=1 << 30, n=1, channels=1, order=16).saved_bytes() == 1 << 36
    assert state_shape(batch=1 << 30, n=1, channels=1, order=16).workspace_bytes() > 1 << 36
    for T in ("float", "half"):
        assert conv_shape(T, n=0).workspace_bytes() == 0 and conv_shape(T, batch=0).workspace_bytes() == 0
        assert conv_shape(T, n=1).workspace_bytes() > 0 and conv_shape(T, n=1, channels=1).workspace_bytes() > 0
    # A sequence at least a part of the taps' and the bias's sums.
    assert conv_shape(batch=8, n=4096, channels=2048).workspace_bytes() < 1 << 24
    assert thff.rms_norm_workspace_bytes(300, 16384) == 4 * 256 * 16384
    assert thff.rms_norm_workspace_bytes(3, 16384) == 4 * 3 * 16384
    assert thff.rms_norm_workspace_bytes(0, 1) == 0 and thff.rms_norm_workspace_bytes(1 << 40, 16385) == 0


@pytest.mark.parametrize("call", [thff.ThunderFFT_short_conv, thff.ThunderFFT_short_conv_async])
def test_conv_refused(call):
    s = conv_shape()
    for x, w, y in ((0, B, D), (A, 0, D), (A, B, 0)):
        with pytest.raises(ValueError, match="non-null"):
            call(s, x, w, C, y)
    for y in (A, B, C, E):
        with pytest.raises(ValueError, match="alias"):
            call(s, A, B, C, y, d_state_in=E)
    for bad in (dict(d_x=A + 1), dict(d_y=D + 1), dict(d_state_in=E + 1), dict(d_state_out=E + 1)):
        args = dict(dict(d_x=A, d_weight=B, d_bias=C, d_y=D), **bad)
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, **args)
    for bad in ("d_weight", "d_bias", "d_slots", "d_lengths"):
        args = dict(dict(d_x=A, d_weight=B, d_bias=C, d_y=D), **{bad: E + 2})
        with pytest.raises(ValueError, match="4-byte aligned"):
            call(s, **args)
    with pytest.raises(ValueError, match="states"):
        call(conv_shape(states=-1), A, B, C, D, d_slots=E)
    with pytest.raises(ValueError, match="non-null"):
        call(conv_shape(n=0), 0, 0, 0, 0, d_state_in=E, d_state_out=E)
    # A shape with nothing to do is done, whatever the pointers.
    call(conv_shape(batch=0), 0, 0, 0, 0)
    call(conv_shape(channels=0), 0, 0, 0, 0)


@pytest.mark.parametrize("call", [thff.ThunderFFT_short_conv_backward, thff.ThunderFFT_short_conv_backward_async])
def test_conv_backward_refused(call):
    s = conv_shape()
    good = dict(d_dy=A, d_x=B, d_weight=C, d_bias=D, d_dx=E, d_dweight=F, d_dbias=G, d_workspace=H)
    for name in ("d_dy", "d_x", "d_weight", "d_dx"):
        with pytest.raises(ValueError, match="non-null"):
            call(s, **dict(good, **{name: 0}))
    with pytest.raises(ValueError, match="requires a workspace"):
        call(s, **dict(good, d_workspace=0))
    for out in ("d_dx", "d_dweight", "d_dbias"):
        for other in ("d_dy", "d_x", "d_weight", "d_bias"):
            with pytest.raises(ValueError, match="alias"):
                call(s, **dict(good, **{out: good[other]}))
    with pytest.raises(ValueError, match="alias"):
        call(s, **dict(good, d_dweight=G))
    with pytest.raises(ValueError, match="alias"):
        call(s, **dict(good, d_dstate_in=9 << 16, d_dstate_out=9 << 16))
    for name in ("d_dy", "d_x", "d_dx", "d_state_in", "d_dstate_out", "d_dstate_in"):
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, **dict(good, **{name: (10 << 16) + 1}))
    for name in ("d_weight", "d_bias", "d_dweight", "d_dbias", "d_lengths"):
        with pytest.raises(ValueError, match="4-byte"):
            call(s, **dict(good, **{name: (10 << 16) + 2}))
    with pytest.raises(ValueError, match="16-byte"):
        call(s, **dict(good, d_workspace=H + 8))
    with pytest.raises(ValueError, match="non-null"):
        call(conv_shape(n=0), 0, 0, 0, 0, 0, d_dstate_in=A, d_dstate_out=B)
    call(conv_shape(channels=0), 0, 0, 0, 0, 0)


@pytest.mark.parametrize("call", [thff.ThunderFFT_state_scan, thff.ThunderFFT_state_scan_async])
def test_state_refused(call):
    s = state_shape()
    good = dict(d_x=A, d_delta=B, d_a=C, d_b=D, d_c=E, d_y=F, d_workspace=G)
    for name in ("d_x", "d_delta", "d_a", "d_b", "d_c", "d_y"):
        with pytest.raises(ValueError, match="non-null"):
            call(s, **dict(good, **{name: 0}))
    for name in ("d_x", "d_delta", "d_a", "d_b", "d_c"):
        with pytest.raises(ValueError, match="alias"):
            call(s, **dict(good, d_y=good[name]))
    for name in ("d_skip", "d_gate", "d_delta_bias", "d_state_in", "d_state_out"):
        with pytest.raises(ValueError, match="alias"):
            call(s, **dict(good, **{name: F}))
    for name in ("d_x", "d_delta", "d_b", "d_c", "d_y", "d_gate"):
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, **dict(good, **{name: H + 1}))
    for name in ("d_a", "d_skip", "d_delta_bias", "d_state_in", "d_state_out", "d_slots", "d_lengths"):
        with pytest.raises(ValueError, match="4-byte aligned"):
            call(s, **dict(good, **{name: H + 2}))
    for name in ("d_saved", "d_workspace"):
        with pytest.raises(ValueError, match="16-byte aligned"):
            call(s, **dict(good, **{name: H + 8}))
    assert s.forward_bytes() > 0
    with pytest.raises(ValueError, match="requires a workspace"):
        call(s, **dict(good, d_workspace=0))
    with pytest.raises(ValueError, match="states must"):
        call(state_shape(states=-1), **dict(good, d_slots=H))
    with pytest.raises(ValueError, match="non-null"):
        call(state_shape(n=0), 0, 0, 0, 0, 0, 0, d_state_in=A, d_state_out=A)
    call(state_shape(batch=0), 0, 0, 0, 0, 0, 0)
    call(state_shape(channels=0, groups=1), 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("call", [thff.ThunderFFT_state_scan_backward, thff.ThunderFFT_state_scan_backward_async])
def test_state_backward_refused(call):
    s = state_shape()
    inputs = ("d_dy", "d_x", "d_delta", "d_a", "d_b", "d_c", "d_saved")
    outputs = ("d_dx", "d_ddelta", "d_da", "d_db", "d_dc")
    good = {name: (k + 1) << 16 for k, name in enumerate(inputs + outputs + ("d_workspace",))}
    other = 40 << 16
    for name in inputs + outputs:
        with pytest.raises(ValueError, match="forward call saved" if name == "d_saved" else "non-null"):
            call(s, **dict(good, **{name: 0}))
    with pytest.raises(ValueError, match="requires a workspace"):
        call(s, **dict(good, d_workspace=0))
    with pytest.raises(ValueError, match="dgate"):
        call(s, **dict(good, d_gate=other))
    for out in outputs:
        for name in inputs + outputs:
            if name != out:
                with pytest.raises(ValueError, match="alias"):
                    call(s, **dict(good, **{out: good[name]}))
    for more in (dict(d_dskip=good["d_x"]), dict(d_gate=other, d_dgate=other), dict(d_ddelta_bias=good["d_da"]),
                 dict(d_dstate_out=other, d_dstate_in=other), dict(d_dskip=other, d_skip=other)):
        with pytest.raises(ValueError, match="alias"):
            call(s, **good, **more)
    for name in ("d_dy", "d_x", "d_delta", "d_b", "d_c", "d_dx", "d_ddelta", "d_db", "d_dc"):
        with pytest.raises(ValueError, match="element-aligned"):
            call(s, **dict(good, **{name: other + 1}))
    for name in ("d_a", "d_skip", "d_delta_bias", "d_dstate_out", "d_lengths", "d_da", "d_dskip", "d_ddelta_bias",
                 "d_dstate_in"):
        with pytest.raises(ValueError, match="4-byte"):
            call(s, **dict(good, **{name: other + 2}))
    for name in ("d_saved", "d_workspace"):
        with pytest.raises(ValueError, match="16-byte"):
            call(s, **dict(good, **{name: other + 4}))
    assert thff.lib().thff_state_scan_backward(s, None, A, 0) == thff.THFF_EINVAL


@pytest.mark.parametrize("twin", ["", "_async"])
def test_rms_refused(twin):
    norm, bits8, backward = (getattr(thff, "ThunderFFT_rms_norm" + name + twin) for name in ("", "_8bit", "_backward"))

    def forward(x=A, weight=B, eps=1e-5, y=C, rows=4, cols=8, T="half", **more):
        norm(T, x, weight, eps, y, rows, cols, **more)

    def quantized(x=A, weight=B, eps=1e-5, q=C, scales=D, rows=4, cols=256, block=128, T="half", **more):
        bits8(T, x, weight, eps, q, scales, rows, cols, block, **more)

    def back(dy=A, total=B, rstd=C, weight=D, dx=E, dweight=0, workspace=0, rows=4, cols=8, T="half", **more):
        backward(T, dy, total, rstd, weight, dx, dweight, workspace, rows, cols, **more)

    for call in (forward, quantized, back):
        with pytest.raises(ValueError, match="float, half and bfloat16"):
            call(T="double")
        for rows, cols, what in ((-1, 8, "rows"), (4, 0, "cols"), (4, -8, "cols"), (4, (1 << 30) + 1, "cols"),
                                 (4, 1 << 32, "out of range")):
            with pytest.raises(ValueError, match=what):
                call(rows=rows, cols=cols)
    for call in (forward, quantized):
        for eps in (-1e-5, float("nan")):
            with pytest.raises(ValueError, match="eps"):
                call(eps=eps)
        for bad, what in ((dict(x=0), "non-null"), (dict(x=C), "alias"), (dict(x=A + 1), "element"), (dict(weight=B + 2), "4-byte"),
                          (dict(d_residual=C), "alias"), (dict(d_residual=E + 1), "element"), (dict(d_sum=A), "alias"),
                          (dict(d_sum=C), "alias"), (dict(d_sum=E + 1), "element"),
                          (dict(d_residual=E, d_sum=E, sum_stride=300), "stride")):
            with pytest.raises(ValueError, match=what):
                call(**bad)
        for stride in ("x_stride", "residual_stride", "sum_stride"):
            with pytest.raises(ValueError, match="stride"):
                call(**{stride: 7})
        call(0, 0, 1e-5, 0, **(dict(scales=0) if call is quantized else {}), rows=0)
    with pytest.raises(ValueError, match="stride"):
        forward(y_stride=7)
    with pytest.raises(ValueError, match="stride"):
        quantized(q_stride=255)
    with pytest.raises(ValueError, match="scales"):
        quantized(scales=0)
    with pytest.raises(ValueError, match="4-byte"):
        quantized(scales=D + 2)
    for block in (0, -1, 64, 255, 512):
        with pytest.raises(ValueError, match="block must be 128 or cols"):
            quantized(block=block)
    with pytest.raises(ValueError, match="4-byte"):
        forward(d_rstd=E + 2)
    for bad, what in ((dict(dy=0), "non-null"), (dict(total=0), "non-null"), (dict(rstd=0), "non-null"), (dict(dx=0), "non-null"),
                      (dict(dy=A + 1), "element"), (dict(total=B + 1), "element"), (dict(dx=E + 1), "element"),
                      (dict(d_dsum=F + 1), "element"), (dict(rstd=C + 2), "4-byte"), (dict(weight=D + 2), "4-byte"),
                      (dict(dx=A), "alias"), (dict(dx=B), "alias"), (dict(d_dsum=E), "alias"), (dict(dweight=D, workspace=H), "alias"),
                      (dict(dweight=F), "requires a workspace"), (dict(dweight=F, workspace=H + 4), "16-byte"),
                      (dict(dy_stride=7), "stride"), (dict(sum_stride=7), "stride"), (dict(dsum_stride=7), "stride"),
                      (dict(dx_stride=7), "stride")):
        with pytest.raises(ValueError, match=what):
            back(**bad)
    back(0, 0, 0, 0, 0, rows=0)  # no rows and no weights


def test_tensor_functions_refuse():
    """There is no CPU path, and shapes are checked."""
    x, a, b = torch.zeros(2, 3, 4), torch.zeros(4, 5), torch.zeros(2, 3, 5)
    for call in (lambda: thff.short_conv(x, torch.zeros(4, 3)), lambda: thff.state_scan(x, x, a, b, b), lambda: thff.rms_norm(x),
                 lambda: thff.rms_norm_8bit(x)):
        with pytest.raises(ValueError, match="device tensor"):
            call()


@pytest.mark.parametrize("name,fields", [("thff_conv_shape", thff.ConvShape._fields_), ("thff_state_shape", thff.StateShape._fields_),
                                         ("thff_state_gradients", thff._StateGradients._fields_)])
def test_c_structs_match(name, fields):
    """The ctypes structs have the C structs' fields, in their order."""
    text = open(os.path.join(os.path.dirname(thff.LIB_PATH), "..", "include", "thunderfft", "thunderfft.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
    assert re.findall(r"(\w+)\s*[,;]", body) == [f[0] for f in fields]
    size = {"thff_conv_shape": 8 * 4 + 2 * 8, "thff_state_shape": 8 * 4 + 6 * 8, "thff_state_gradients": 21 * 8}[name]
    kind = {"thff_conv_shape": thff.ConvShape, "thff_state_shape": thff.StateShape, "thff_state_gradients": thff._StateGradients}[name]
    assert ctypes.sizeof(kind) == size


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


def against_differences(values, outputs, grads, names):
    """Gradients along random directions against central differences of the same sums in 64 bits: a
    step of 2^-17 leaves a truncation of 2^-34 of the third derivatives and a rounding of
    2^-53 / 2^-17 of the sums, both far below 1e-6 of sums of order a hundred."""
    eps, gen = 2.0 ** -17, torch.Generator().manual_seed(9)
    for at, name in enumerate(names):
        v = normal(gen, *values[at].shape)
        up, down = list(values), list(values)
        up[at], down[at] = values[at] + eps * v, values[at] - eps * v
        along = float((grads[name][0] * v.view(grads[name][0].shape)).sum())
        assert abs((outputs(*up) - outputs(*down)) / (2 * eps) - along) < 1e-6, name


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("silu", [True, False])
def test_conv_oracle_gradients(width, silu):
    gen = torch.Generator().manual_seed(5)
    values = [normal(gen, 3, 7, 5), normal(gen, 5, width), normal(gen, 5), normal(gen, 3, width - 1, 5)]
    dy, dstate, lengths = normal(gen, 3, 7, 5), normal(gen, 3, width - 1, 5), torch.tensor([7, 1, 0])
    got = oracle.conv("float", *values, lengths, silu, dy, dstate)

    def outputs(*v):
        r = oracle.conv("float", *v, lengths, silu)
        return float((r["y"][0] * dy).sum() + (r["state"][0] * dstate).sum())

    against_differences(values, outputs, got, ("dx", "dweight", "dbias", "dstate"))


@pytest.mark.parametrize("gated", [True, False])
def test_state_oracle_gradients(gated):
    gen = torch.Generator().manual_seed(6)
    batch, n, channels, order, groups = 3, 6, 4, 3, 2
    values = [normal(gen, batch, n, channels), normal(gen, batch, n, channels), -normal(gen, channels, order).exp(),
              normal(gen, batch, n, groups, order), normal(gen, batch, n, groups, order), normal(gen, channels),
              normal(gen, batch, n, channels), normal(gen, channels), normal(gen, batch, channels, order)]
    dy, dstate, lengths = normal(gen, batch, n, channels), normal(gen, batch, channels, order), torch.tensor([6, 4, 0])

    def call(*v, **more):
        v = list(v)
        if not gated:
            v[6] = None
        return oracle.state("float", *v, lengths, **more)

    def outputs(*v):
        r = call(*v)
        return float((r["y"][0] * dy).sum() + (r["state"][0] * dstate).sum())

    names = ["dx", "ddelta", "da", "db", "dc", "dskip", "dgate", "ddelta_bias", "dstate"]
    got = call(*values, dy=dy, dstate=dstate)
    if not gated:
        got["dgate"] = (torch.zeros_like(values[6]), None)
    against_differences(values, outputs, got, names)


def test_rms_oracle_gradients():
    gen = torch.Generator().manual_seed(7)
    values = [normal(gen, 4, 7), normal(gen, 7)]
    dy, dsum, residual = normal(gen, 4, 7), normal(gen, 4, 7), normal(gen, 4, 7)
    got = oracle.rms("float", values[0], values[1], 1e-5, residual, dy, dsum)

    def outputs(x, w):
        r = oracle.rms("float", x, w, 1e-5, residual)
        return float((r["y"][0] * dy).sum() + (r["sum"][0] * dsum).sum())

    against_differences(values, outputs, got, ("dx", "dweight"))


@pytest.mark.parametrize("twin", ["", "_async"])
def test_outputs_in_another_arrays_place(twin):
    """States, statistics and scratch memory that a call writes are no other array's: kept in place are only
    states (state_out = state_in) and residuals."""
    def refused(call, **arrays):
        with pytest.raises(ValueError, match="alias"):
            call(**arrays)

    conv, scan, norm, bits8 = (getattr(thff, f"ThunderFFT_{name}{twin}") for name in ("short_conv", "state_scan", "rms_norm", "rms_norm_8bit"))
    good = dict(shape=conv_shape(), d_x=A, d_weight=B, d_bias=C, d_y=D, d_slots=E, d_lengths=F)
    for name in ("d_x", "d_weight", "d_bias", "d_y", "d_slots", "d_lengths"):
        refused(conv, **good, d_state_out=good[name])
    for name in ("d_slots", "d_lengths"):
        refused(conv, **dict(good, d_y=good[name]))
    refused(conv, **dict(good, shape=conv_shape(n=0), d_state_out=B))
    more = 9 << 16
    good = dict(shape=state_shape(), d_x=A, d_delta=B, d_a=C, d_b=D, d_c=E, d_y=F, d_skip=G, d_gate=H, d_delta_bias=more,
                d_state_in=more << 1, d_slots=more << 2, d_lengths=more << 3, d_saved=more << 4, d_workspace=more << 5)
    for name in good:
        if name not in ("shape", "d_state_in"):
            refused(scan, **good, d_state_out=good[name])
        if name not in ("shape", "d_saved", "d_workspace"):
            refused(scan, **dict(good, d_saved=good[name]))
            refused(scan, **dict(good, d_workspace=good[name]))
    refused(scan, **dict(good, d_saved=more << 5))
    refused(norm, T="half", d_x=A, d_weight=B, eps=1e-5, d_y=C, rows=4, cols=8, d_residual=E, d_rstd=E)
    refused(bits8, T="half", d_x=A, d_weight=B, eps=1e-5, d_q=C, d_scales=E, rows=4, cols=256, d_residual=E)

    back = getattr(thff, "ThunderFFT_short_conv_backward" + twin)
    good = dict(shape=conv_shape(), d_dy=A, d_x=B, d_weight=C, d_bias=D, d_dx=E, d_dweight=F, d_dbias=G, d_lengths=more, d_workspace=H)
    for name in good:
        if name not in ("shape", "d_workspace"):
            refused(back, **dict(good, d_workspace=good[name]))
    refused(back, **dict(good, d_dweight=more))
    back = getattr(thff, "ThunderFFT_state_scan_backward" + twin)
    names = ("d_dy", "d_x", "d_delta", "d_a", "d_b", "d_c", "d_saved", "d_dx", "d_ddelta", "d_da", "d_db", "d_dc", "d_lengths")
    good = dict({name: (k + 1) << 16 for k, name in enumerate(names)}, shape=state_shape())
    for name in names:
        refused(back, **good, d_workspace=good[name])
    refused(back, **dict(good, d_da=good["d_lengths"], d_workspace=more << 8))
    back = getattr(thff, "ThunderFFT_rms_norm_backward" + twin)
    good = dict(T="half", d_dy=A, d_sum=B, d_rstd=C, d_weight=D, d_dx=E, d_dweight=F, d_dsum=G, rows=4, cols=8)
    for name in ("d_dy", "d_sum", "d_rstd", "d_weight", "d_dx", "d_dweight", "d_dsum"):
        refused(back, **good, d_workspace=good[name])


class OnDevice:
    """Stands for a tensor on the device at `at`."""

    def __init__(self, t, at):
        self.dtype, self.is_cuda, self.is_contiguous, self.stride, self.at = t.dtype, True, t.is_contiguous, t.stride, at

    def data_ptr(self):
        return self.at


def test_slots_and_lengths_refused(monkeypatch):
    """Tensors in host memory, of another type or with gaps: kernels would index by what they read there."""
    given = []
    monkeypatch.setattr(thff, "_raise", lambda rc: given.append(rc))
    good = torch.zeros(8, dtype=torch.int32)
    wrong = ((good, "device memory"), (OnDevice(good.long(), G), "int32"), (OnDevice(good.float(), G), "int32"),
             (OnDevice(good[::2], G), "gaps"), (OnDevice(good.view(4, 2)[:, 0], G), "gaps"))
    scan = thff.ScanShape("half", 2, 300, 70)
    args = dict.fromkeys(("d_dy", "d_x", "d_delta", "d_a", "d_b", "d_c", "d_saved", "d_dx", "d_ddelta", "d_da", "d_db", "d_dc"), 0)
    both = (("d_slots", "d_lengths"), lambda **more: thff.ThunderFFT_short_conv_async(conv_shape(), 0, B, C, D, **more)), (
        ("d_slots", "d_lengths"), lambda **more: thff.ThunderFFT_state_scan_async(state_shape(), 0, B, C, D, E, F, **more)), (
        ("d_slots", "d_lengths"), lambda **more: thff.ThunderFFT_gated_scan_async(scan, 0, B, C, **more)), (
        ("d_lengths",), lambda **more: thff.ThunderFFT_short_conv_backward_async(conv_shape(), 0, B, C, D, E, F, G, **more)), (
        ("d_lengths",), lambda **more: thff.ThunderFFT_state_scan_backward_async(state_shape(), **args, **more)), (
        ("d_lengths",), lambda **more: thff.ThunderFFT_gated_scan_backward_async(scan, 0, B, C, D, E, F, **more))
    for names, call in both:
        for name in names:
            for t, what in wrong:
                with pytest.raises(ValueError, match=what):
                    call(**{name: t})
            given.clear()
            # These reach the library, which refuses the null pointers beside them.
            for t in (None, G, OnDevice(good, G), OnDevice(good.view(8, 1)[:, 0], G)):
                call(**{name: t})
            assert given == [thff.THFF_EINVAL] * 4


def test_arrays_of_no_bytes_lie_anywhere(monkeypatch):
    """Scratch memory that a call does not use, and arrays of no steps, may have the address of what follows them."""
    monkeypatch.setattr(thff, "_raise", lambda rc: given.append(rc))
    given = []
    one = state_shape(n=1)
    assert one.forward_bytes() == 0 and thff.rms_norm_workspace_bytes(4, 20000) == 0
    # The last argument is off its alignment, which is looked at after the addresses.
    for call, args in (
            (thff.ThunderFFT_state_scan, dict(shape=one, d_x=A, d_delta=B, d_a=C, d_b=D, d_c=E, d_y=F, d_workspace=F, d_skip=G + 2)),
            (thff.ThunderFFT_state_scan, dict(shape=state_shape(n=0), d_x=A, d_delta=A, d_a=C, d_b=A, d_c=A, d_y=A, d_state_out=A,
                                              d_workspace=A, d_skip=G + 2)),
            (thff.ThunderFFT_short_conv, dict(shape=conv_shape(n=0), d_x=A, d_weight=C, d_bias=D + 2, d_y=A, d_state_out=A)),
            (thff.ThunderFFT_short_conv_backward, dict(shape=conv_shape(), d_dy=A, d_x=B, d_weight=C, d_bias=D + 2, d_dx=E,
                                                       d_workspace=E)),
            (thff.ThunderFFT_short_conv_backward, dict(shape=conv_shape(n=0), d_dy=A, d_x=A, d_weight=C, d_bias=D + 2, d_dx=A,
                                                       d_dweight=A, d_dstate_in=E)),
            (thff.ThunderFFT_state_scan_backward, dict(shape=state_shape(n=0), d_dy=A, d_x=A, d_delta=A, d_a=C, d_b=A, d_c=A,
                                                       d_saved=A, d_dx=A, d_ddelta=A, d_da=A, d_db=A, d_dc=A, d_skip=G + 2,
                                                       d_workspace=B)),
            (thff.ThunderFFT_rms_norm_backward, dict(T="half", d_dy=A, d_sum=B, d_rstd=C, d_weight=D + 2, d_dx=E, d_dweight=F,
                                                     d_workspace=A, rows=4, cols=20000))):
        given.clear()
        call(**args)
        assert given == [thff.THFF_EINVAL] and b"4-byte aligned" in thff.lib().thff_last_error(), (call.__name__, thff.lib().thff_last_error())
