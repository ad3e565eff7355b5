"""The gated linear recurrence on the GPU against its definition in 64 bits: outputs, final
states and gradients, in both layouts and all types, from lengths of zero to thousands, with
the strides, masks, slots and streams that a program uses."""
import itertools

import pytest
import torch

import sequence_oracle as oracle
import thunderfft_amd as thff

pytestmark = pytest.mark.gpu
LAYOUTS = ("channels_last", "channels_first")
GUARD = -271.0


def values(seed, T, layout, batch, n, channels, fused=False, offset=0):
    """x, gate, dy, state, dstate on the GPU.  fused: x and the gate side by side in rows;
    offset: elements between the buffers' aligned start and the first value."""
    gen = torch.Generator().manual_seed(seed)
    dims = (batch, n, channels) if layout == "channels_last" else (batch, channels, n)

    def normal(*s, mean=0.0, std=1.0):
        return torch.randn(*s, generator=gen) * std + mean

    def placed(v):
        whole = torch.full((v.numel() + offset,), GUARD, dtype=oracle.TYPES[T], device="cuda")
        part = whole[offset:].view(v.shape)
        part.copy_(v)
        return part

    x, gate, dy = placed(normal(*dims)), placed(normal(*dims, mean=1.5, std=2.5)), placed(normal(*dims))
    if fused:
        both = placed(torch.cat([x.cpu().float(), gate.cpu().float()], -1))
        x, gate = both[..., :dims[-1]], both[..., dims[-1]:]
    return x, gate, dy, normal(batch, channels).cuda(), normal(batch, channels).cuda()


def shape_of(T, layout, x, gate, **more):
    batch, n, channels = x.shape if layout == "channels_last" else (x.shape[0], x.shape[2], x.shape[1])
    stride = x.stride(1) if x.shape[1] > 1 or x.shape[0] == 1 else x.stride(0)
    return thff.ScanShape(T, batch, n, channels, layout=layout, x_stride=max(stride, x.shape[2]),
                          gate_stride=max(stride, x.shape[2]), **more)


def buffers(s):
    saved = torch.full((s.saved_bytes(),), 0xFF, dtype=torch.uint8, device="cuda")
    workspace = torch.full((s.workspace_bytes(),), 0xFF, dtype=torch.uint8, device="cuda")
    return saved, workspace


def guarded(dims, stride, dtype, offset=0):
    """An output whose rows lie `stride` apart, and whether what is around them is as it was."""
    rows, cols = dims[0] * dims[1], dims[2]
    whole = torch.full((offset + rows * stride + 64,), GUARD, dtype=dtype, device="cuda")
    out = whole[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    out.fill_(float("nan"))

    def intact():
        around = whole.clone()
        around[offset:offset + rows * stride].view(rows, stride)[:, :cols] = GUARD
        return bool((around == GUARD).all())

    return out.unflatten(0, dims[:2]), intact


def run(T, layout, x, gate, dy, state, dstate, lengths=None, gap=0, offset=0, with_state=True):
    """Forward and backward pass into guarded outputs; {name: tensor}."""
    s = shape_of(T, layout, x, gate, y_stride=x.shape[2])
    saved, workspace = buffers(s)
    dt = x.dtype
    y, y_ok = guarded(x.shape, x.shape[2] + gap, dt, offset)
    last, last_ok = guarded((1, s.batch, s.channels), s.channels, torch.float32)
    s.y_stride = x.shape[2] + gap
    print(f"{T} {layout} {tuple(x.shape)} stride {s.x_stride} gap {gap} offset {offset}", flush=True)
    state = state if with_state else None
    thff.ThunderFFT_gated_scan(s, x, gate, y, d_state_in=state, d_state_out=last, d_lengths=lengths,
                               d_saved=saved, d_workspace=workspace)
    assert y_ok() and last_ok()
    # The gradients have the strides of what they are gradients of.
    if s.x_stride == 2 * x.shape[2]:
        both, in_ok = guarded((*x.shape[:2], 2 * x.shape[2]), 2 * x.shape[2], dt, offset)
        dx, dgate = both[..., :x.shape[2]], both[..., x.shape[2]:]
        gate_ok = in_ok
    else:
        dx, in_ok = guarded(x.shape, s.x_stride, dt, offset)
        dgate, gate_ok = guarded(x.shape, s.x_stride, dt, offset)
    dfirst, first_ok = guarded((1, s.batch, s.channels), s.channels, torch.float32)
    if gap:
        wide, _ = guarded(x.shape, s.y_stride, dt, offset)
        wide.copy_(dy)
        dy = wide
    else:
        dy = dy.contiguous()
    thff.ThunderFFT_gated_scan_backward(s, dy, x, gate, saved, dx, dgate,
                                        d_dstate_out=dstate if with_state else None, d_dstate_in=dfirst,
                                        d_lengths=lengths, d_workspace=workspace)
    assert in_ok() and gate_ok() and first_ok()
    return dict(y=y, state=last[0], dx=dx, dgate=dgate, dstate=dfirst[0])


def compare(T, layout, x, gate, dy, state, dstate, lengths=None, with_state=True, **how):
    got = run(T, layout, x, gate, dy, state, dstate, lengths, with_state=with_state, **how)
    want = oracle.scan(T, layout, x, gate, state if with_state else None, lengths, dy,
                       dstate if with_state else None)
    for name in want:
        oracle.check(name, got[name], want[name])


# Sizes on both sides of whatever a kernel takes at once: lanes, vectors, steps of a wave, of
# a workgroup and of several.
SIZES = [(1, 1, 1), (3, 1, 130), (2, 2, 7), (1, 15, 64), (2, 16, 66), (1, 17, 8), (2, 63, 128), (1, 64, 129),
         (3, 127, 40), (1, 128, 256), (2, 129, 24), (1, 255, 130), (1, 257, 65), (1, 511, 16), (2, 513, 2),
         (1, 1000, 200), (1, 1025, 72), (1, 2047, 4), (1, 2049, 33), (2, 4100, 10), (1, 8200, 3)]


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(T, layout, size):
    compare(T, layout, *values(sum(size), T, layout, *size))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("how", [dict(gap=1), dict(gap=8), dict(offset=1), dict(offset=2), dict(offset=8, gap=24),
                                 dict(fused=True), dict(fused=True, offset=3), dict(with_state=False)], ids=str)
def test_strides_and_offsets(T, layout, how):
    """Rows with gaps, buffers off the 16-byte boundary, halves of one projection, no state."""
    for size in ((2, 130, 72), (1, 300, 136), (3, 40, 37)):
        more = dict(how)
        fused, offset = more.pop("fused", False), more.get("offset", 0)
        compare(T, layout, *values(7, T, layout, *size, fused=fused, offset=offset), **more)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
def test_lengths(T, layout):
    """Sequences that end early, at once, or never; what lies past the end is NaN, infinite
    or the type's lowest value in x, the gate and dy, and reaches nothing."""
    lengths = [0, 1, 15, 16, 100, 128, 129, 255, 256, 299, 300, 400, -3]
    batch, n, channels = len(lengths), 300, 70
    x, gate, dy, state, dstate = values(11, T, layout, batch, n, channels)
    on = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    past = torch.arange(n, device="cuda") >= on.unsqueeze(1)
    past = past.unsqueeze(2) if layout == "channels_last" else past.unsqueeze(1)
    for v, junk in ((x, float("nan")), (gate, float("inf")), (dy, torch.finfo(dy.dtype).min)):
        v.masked_fill_(past, junk)
    compare(T, layout, x, gate, dy, state, dstate, on.clamp(0, n))
    # Outside [0, n] is taken to the nearer end.
    within = run(T, layout, x, gate, dy, state, dstate, on.clamp(0, n))
    outside = run(T, layout, x, gate, dy, state, dstate, on)
    for name in within:
        assert torch.equal(within[name], outside[name]), name


@pytest.mark.parametrize("T", ["float", "half"])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_short_lengths_of_long_rows(T, layout):
    """Most of the steps are padding: states and gradients pass over it unchanged."""
    lengths = torch.tensor([0, 1, 130, 9000, 4700], dtype=torch.int32, device="cuda")
    x, gate, dy, state, dstate = values(15, T, layout, len(lengths), 9000, 18)
    compare(T, layout, x, gate, dy, state, dstate, lengths)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_no_steps(layout):
    """n = 0 hands the states through, also by slots."""
    s = thff.ScanShape("half", 3, 0, 130, layout=layout, states=5)
    state, last = torch.randn(5, 130).cuda(), torch.full((5, 130), GUARD).cuda()
    slots = torch.tensor([4, -1, 0], dtype=torch.int32).cuda()
    thff.ThunderFFT_gated_scan(s, 0, 0, 0, d_state_in=state, d_state_out=last, d_slots=slots)
    assert torch.equal(last[4], state[4]) and torch.equal(last[0], state[0])
    assert (last[1:4] == GUARD).all()
    back = torch.full((3, 130), GUARD).cuda()
    thff.ThunderFFT_gated_scan_backward(s, 0, 0, 0, 0, 0, 0, d_dstate_out=state, d_dstate_in=back)
    assert torch.equal(back, state[:3])
    thff.ThunderFFT_gated_scan(s, 0, 0, 0, d_state_out=last)
    assert (last[:3] == 0).all()


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [1, 5, 200])
def test_slots(T, layout, n):
    """States in a pool by slot; empty places (outside the pool) start from zero and store
    nothing; other rows of the pool stay as they are; in place and into another pool."""
    batch, channels, rows = 6, 136, 9
    x, gate, _, _, _ = values(3, T, layout, batch, n, channels)
    pool = torch.randn(rows, channels).cuda()
    slots = torch.tensor([8, -1, 0, 9, 3, 2 ** 31 - 1], dtype=torch.int32).cuda()
    empty = (slots < 0) | (slots >= rows)
    state = torch.where(empty.unsqueeze(1), 0.0, pool[slots.clamp(0, rows - 1).long()])
    want = oracle.scan(T, layout, x, gate, state)
    s = shape_of(T, layout, x, gate, states=rows)
    _, workspace = buffers(s)
    for out in (torch.full_like(pool, GUARD), pool.clone()):
        y = torch.empty_like(x)
        before, into = (pool, out) if float(out[0, 0]) == GUARD else (out, out)
        untouched = into.clone()
        thff.ThunderFFT_gated_scan(s, x, gate, y, d_state_in=before, d_state_out=into, d_slots=slots,
                                   d_workspace=workspace)
        oracle.check("y", y, want["y"])
        value, bound = want["state"]
        keep = [i for i in range(batch) if not bool(empty[i])]
        oracle.check("state", into[slots[keep].long()], (value[keep], bound[keep]))
        rest = [r for r in range(rows) if r not in slots[keep].tolist()]
        assert torch.equal(into[rest], untouched[rest])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
def test_token_by_token(T, layout):
    """A prompt and then single tokens in place give what one call over all steps gives."""
    batch, n, channels, prompt = 3, 40, 136, 33
    x, gate, _, state, _ = values(4, T, layout, batch, n, channels)
    want = oracle.scan(T, layout, x, gate, state)
    axis = 1 if layout == "channels_last" else 2
    held = state.clone()
    parts = []
    for lo, hi in [(0, prompt)] + [(t, t + 1) for t in range(prompt, n)]:
        px, pg = x.narrow(axis, lo, hi - lo).contiguous(), gate.narrow(axis, lo, hi - lo).contiguous()
        s = shape_of(T, layout, px, pg)
        y = torch.empty_like(px)
        thff.ThunderFFT_gated_scan(s, px, pg, y, d_state_in=held, d_state_out=held,
                                   d_workspace=buffers(s)[1])
        parts.append(y)
    oracle.check("y", torch.cat(parts, axis), want["y"])
    oracle.check("state", held, want["state"])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_extreme_gates(layout):
    """Gates of the type's ends keep or replace the state exactly; infinite ones too."""
    for T in oracle.TYPES:
        x, gate, _, state, _ = values(5, T, layout, 2, 50, 24)
        for g in (torch.finfo(gate.dtype).max, float("inf")):
            s = shape_of(T, layout, x, gate)
            for sign in (1, -1):
                y = torch.empty_like(x)
                thff.ThunderFFT_gated_scan(s, x, torch.full_like(gate, sign * g), y, d_state_in=state,
                                           d_workspace=buffers(s)[1])
                held = state.to(x.dtype).unsqueeze(1 if layout == "channels_last" else 2).expand_as(x)
                assert torch.equal(y, held if sign > 0 else x), (T, g, sign)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_values_stay_in_their_sequence(layout, bad):
    """A NaN or infinity makes the later outputs of its sequence and channel non-finite, and
    changes no other bit."""
    x, gate, _, state, _ = values(6, "bfloat16", layout, 3, 700, 40)
    s = shape_of("bfloat16", layout, x, gate)
    workspace = buffers(s)[1]

    def call():
        y = torch.empty_like(x)
        thff.ThunderFFT_gated_scan(s, x, gate, y, d_state_in=state, d_workspace=workspace)
        return y

    clean = call()
    at = (1, 333, 21) if layout == "channels_last" else (1, 21, 333)
    x[at] = bad
    got = call()
    later = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    if layout == "channels_last":
        later[1, 333:, 21] = True
    else:
        later[1, 21, 333:] = True
    assert torch.equal(got[~later], clean[~later])
    assert not torch.isfinite(got[later]).any()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_infinite_values_stay_infinite(layout):
    """A state that has overflowed keeps its sign to the end, however many gates, all above zero,
    have been multiplied since; so does a gradient to the first step."""
    x, gate, dy, state, _ = values(12, "half", layout, 2, 9000, 6)
    axis = 1 if layout == "channels_last" else 2
    first, last = x.narrow(axis, 3, 1), dy.narrow(axis, 8990, 1)
    first.copy_(torch.where(first > 0, float("inf"), -float("inf")))
    last.copy_(torch.where(last > 0, float("inf"), -float("inf")))
    got = run("half", layout, x, gate, dy, state, None, with_state=False)
    assert torch.equal(got["y"].narrow(axis, 3, 8997), first.expand(x.shape).narrow(axis, 3, 8997))
    assert torch.isfinite(got["y"].narrow(axis, 0, 3)).all()
    assert torch.equal(got["dx"].narrow(axis, 0, 8991), last.expand(x.shape).narrow(axis, 0, 8991))
    assert torch.isfinite(got["dx"].narrow(axis, 8991, 9)).all()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_same_bits_each_time(layout):
    """Calls repeat to the bit, whatever the workspace held and whatever runs beside them."""
    x, gate, dy, state, dstate = values(8, "bfloat16", layout, 2, 6000, 130)
    first = run("bfloat16", layout, x, gate, dy, state, dstate)
    for _ in range(5):
        again = run("bfloat16", layout, x, gate, dy, state, dstate)
        for name in first:
            assert torch.equal(first[name], again[name]), name


@pytest.mark.parametrize("layout", LAYOUTS)
def test_streams_do_not_meet(layout):
    """Calls on several streams at once, each with its own buffers, as one after the other."""
    sets = [values(20 + k, "half", layout, 2, 3000, 96) for k in range(3)]
    alone = [run("half", layout, *v) for v in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    shapes = [shape_of("half", layout, v[0], v[1]) for v in sets]
    spaces = [buffers(s) for s in shapes]
    outs = [torch.empty_like(v[0]) for v in sets]
    grads = [(torch.empty_like(v[0]), torch.empty_like(v[0])) for v in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        for (x, gate, dy, state, dstate), st, s, (saved, ws), y, (dx, dg) in zip(sets, streams, shapes, spaces, outs, grads):
            thff.ThunderFFT_gated_scan_async(s, x, gate, y, d_state_in=state, d_saved=saved, d_workspace=ws, stream=st)
            thff.ThunderFFT_gated_scan_backward_async(s, dy, x, gate, saved, dx, dg, d_dstate_out=dstate,
                                                      d_workspace=ws, stream=st)
    torch.cuda.synchronize()
    for want, y, (dx, dg) in zip(alone, outs, grads):
        assert torch.equal(want["y"], y) and torch.equal(want["dx"], dx) and torch.equal(want["dgate"], dg)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("size", [(4, 1, 136), (2, 3000, 96)], ids=str)
def test_graph_replays(layout, size):
    """Captured and replayed with new inputs, eager calls in between; every replay is checked."""
    x, gate, dy, state, dstate = values(30, "bfloat16", layout, *size)
    s = shape_of("bfloat16", layout, x, gate)
    saved, workspace = buffers(s)
    y, dx, dg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)

    def calls(stream):
        thff.ThunderFFT_gated_scan_async(s, x, gate, y, d_state_in=state, d_saved=saved, d_workspace=workspace,
                                         stream=stream)
        thff.ThunderFFT_gated_scan_backward_async(s, dy, x, gate, saved, dx, dg, d_dstate_out=dstate,
                                                  d_workspace=workspace, stream=stream)

    calls(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for k in range(4):
        new = values(40 + k, "bfloat16", layout, *size)
        for old, v in zip((x, gate, dy, state, dstate), new):
            old.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = run("bfloat16", layout, *new)
        assert torch.equal(want["y"], y) and torch.equal(want["dx"], dx) and torch.equal(want["dgate"], dg), k


@pytest.mark.parametrize("layout", LAYOUTS)
def test_offsets_past_32_bits(layout):
    """Rows so far apart that the last lie over 2^32 elements from the first."""
    batch, n, channels = (1, 5, 40) if layout == "channels_last" else (1, 5, 6)
    rows, stride = (5, (1 << 30) + 8) if layout == "channels_last" else (6, 1 << 30)
    x, gate, dy, state, dstate = values(9, "half", layout, batch, n, channels)
    base = torch.empty((rows - 1) * stride + 512, dtype=torch.float16, device="cuda")
    far = [base.as_strided(x.shape, (rows * stride, stride, 1), 64 * k) for k in range(6)]
    for f, v in zip(far, (x, gate, dy)):
        f.copy_(v)
    s = thff.ScanShape("half", batch, n, channels, layout=layout, x_stride=stride, gate_stride=stride, y_stride=stride)
    saved, workspace = buffers(s)
    last, dfirst = torch.empty(batch, channels, device="cuda"), torch.empty(batch, channels, device="cuda")
    thff.ThunderFFT_gated_scan(s, far[0], far[1], far[3], d_state_in=state, d_state_out=last, d_saved=saved,
                               d_workspace=workspace)
    want = oracle.scan("half", layout, x, gate, state, None, dy, dstate)
    oracle.check("y", far[3], want["y"])
    thff.ThunderFFT_gated_scan_backward(s, far[2], far[0], far[1], saved, far[4], far[5], d_dstate_out=dstate,
                                        d_dstate_in=dfirst, d_workspace=workspace)
    for name, v in (("state", last), ("dx", far[4]), ("dgate", far[5]), ("dstate", dfirst)):
        oracle.check(name, v, want[name])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_gradients_against_differences(layout):
    """The float gradients along a direction against a central difference of the float
    forward pass: off by its roundings over the step, and by the truncation, which the same
    quotient in 64 bits has."""
    x, gate, dy, state, dstate = values(12, "float", layout, 2, 200, 24)
    got = run("float", layout, x, gate, dy, state, dstate)
    s = shape_of("float", layout, x, gate)
    workspace = buffers(s)[1]
    eps = 2.0 ** -8

    def losses(ins):
        y, last = torch.empty_like(x), torch.empty_like(state)
        thff.ThunderFFT_gated_scan(s, ins[0], ins[1], y, d_state_in=ins[2], d_state_out=last, d_workspace=workspace)
        here = float((y.double() * dy.double()).sum() + (last.double() * dstate.double()).sum())
        w = oracle.scan("float", layout, *ins)
        there = float((w["y"][0] * dy.cpu().double()).sum() + (w["state"][0] * dstate.cpu().double()).sum())
        off = float((w["y"][1] * dy.cpu().double().abs()).sum() + (w["state"][1] * dstate.cpu().double().abs()).sum())
        return here, there, off

    want = oracle.scan("float", layout, x, gate, state, None, dy, dstate)
    gen = torch.Generator().manual_seed(1)
    for name, at in (("dx", 0), ("dgate", 1), ("dstate", 2)):
        ins = [x, gate, state]
        v = torch.randn(ins[at].shape, generator=gen).cuda()
        up, down = list(ins), list(ins)
        up[at], down[at] = ins[at] + eps * v, ins[at] - eps * v
        step = (up[at].double() - down[at].double()).cpu()  # the step as it is in float
        a, b = losses(up), losses(down)
        quotient, exact = a[0] - b[0], a[1] - b[1]
        along = float((got[name].cpu().double() * step).sum())
        truncation = abs(exact - float((want[name][0] * step).sum()))
        bound = a[2] + b[2] + truncation + float((want[name][1] * step.abs()).sum())
        assert abs(quotient - along) <= bound, (name, quotient, along, bound)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
def test_tensor_function(T, layout):
    """gated_scan with its gradients, on halves of a projection, and on another stream."""
    x, gate, dy, state, dstate = values(13, T, layout, 3, 150, 40, fused=True)
    lengths = torch.tensor([150, 0, 77], dtype=torch.int32).cuda()
    leaves = [v.clone() if v is state else v for v in (x, gate, state)]
    leaves = [v.detach().requires_grad_() for v in leaves]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y, last = thff.gated_scan(*leaves, lengths=lengths, layout=layout)
        torch.autograd.backward([y, last], [dy, dstate])
    stream.synchronize()
    want = oracle.scan(T, layout, x, gate, state, lengths, dy, dstate)
    for name, v in (("y", y), ("state", last), ("dx", leaves[0].grad), ("dgate", leaves[1].grad),
                    ("dstate", leaves[2].grad)):
        oracle.check(name, v, want[name])
    # Without a state, without gradients, and only the last state used.
    y2, last2 = thff.gated_scan(x, gate, layout=layout)
    assert not y2.requires_grad
    only = gate.detach().clone().requires_grad_()
    _, last3 = thff.gated_scan(x, only, layout=layout)
    last3.backward(dstate)
    want = oracle.scan(T, layout, x, gate, None, None, torch.zeros_like(x), dstate)
    oracle.check("dgate", only.grad, want["dgate"])
    oracle.check("state", last2, want["state"])


def test_tensor_function_refuses():
    x = torch.zeros(2, 3, 4, device="cuda")
    for bad in (dict(gate=x[:, :2]), dict(gate=x.half()), dict(gate=x.cpu()), dict(state=torch.zeros(2, 3, device="cuda")),
                dict(state=torch.zeros(2, 4, device="cuda", dtype=torch.float16)),
                dict(lengths=torch.zeros(2, device="cuda")), dict(lengths=torch.zeros(3, device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            thff.gated_scan(**{"x": x, "gate": x, **bad})
    with pytest.raises(ValueError):
        thff.gated_scan(x.double(), x.double())
    with pytest.raises(ValueError):
        thff.gated_scan(x[0], x[0])


def test_empty_tensors():
    for dims in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        for layout in LAYOUTS:
            x = torch.zeros(dims, device="cuda", requires_grad=True)
            channels = dims[2] if layout == "channels_last" else dims[1]
            state = torch.ones(dims[0], channels, device="cuda", requires_grad=True)
            y, last = thff.gated_scan(x, x, state, layout=layout)
            assert y.shape == x.shape and last.shape == state.shape
            steps = dims[1] if layout == "channels_last" else dims[2]
            if steps == 0:
                assert torch.equal(last, state)
            (y.sum() + last.sum()).backward()
            if steps == 0:
                assert torch.equal(state.grad, torch.ones_like(state))


@pytest.mark.parametrize("seed", range(24))
def test_drawn(seed):
    """Shapes over the whole range, as programs have them."""
    import random

    rng = random.Random(seed)
    T, layout = rng.choice(list(oracle.TYPES)), LAYOUTS[seed % 2]
    n = int(2 ** rng.uniform(0, 13.5))
    channels = max(1, min(int(2 ** rng.uniform(0, 11)), (1 << 19) // n))
    batch = max(1, min(rng.randint(1, 9), (1 << 19) // (n * channels)))
    lengths = None
    if rng.random() < 0.5:
        lengths = torch.tensor([rng.randint(0, n) for _ in range(batch)], dtype=torch.int32).cuda()
    fused, offset, gap = rng.random() < 0.4, rng.choice([0, 0, 1, 4]), rng.choice([0, 0, 3, 8])
    compare(T, layout, *values(seed, T, layout, batch, n, channels, fused=fused, offset=offset), lengths,
            gap=gap, offset=offset)


@pytest.mark.parametrize("T", ["float", "bfloat16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("size", [(1, 7400, 64), (2, 9000, 65), (1, 33000, 5)], ids=str)
def test_few_channels_and_many_steps(T, layout, size):
    """Chains of tens to hundreds of tiles, one or a few side by side."""
    compare(T, layout, *values(sum(size), T, layout, *size))


def test_long_sequences():
    """More steps than any workgroup keeps, few channels: the state is carried a long way
    (nearly closed gates), against the definition."""
    for layout, T in itertools.product(LAYOUTS, ("float", "bfloat16")):
        x, gate, dy, state, dstate = values(14, T, layout, 1, 30011, 6)
        gate += 6
        compare(T, layout, x, gate, dy, state, dstate)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [1, 700, 9000])
def test_states_in_place(layout, n):
    """The last state may go where the first one was, also where many workgroups share a row and a
    sequence ends in the first of them."""
    x, gate, _, state, _ = values(14, "bfloat16", layout, 4, n, 70)
    s = shape_of("bfloat16", layout, x, gate)
    lengths = torch.tensor([n, n // 2, 3, 0], dtype=torch.int32).clamp(max=n).cuda()
    out, apart, inplace, y = torch.empty_like(state), torch.empty_like(x), state.clone(), torch.empty_like(x)
    thff.ThunderFFT_gated_scan(s, x, gate, apart, d_state_in=state, d_state_out=out, d_lengths=lengths,
                               d_workspace=buffers(s)[1])
    thff.ThunderFFT_gated_scan(s, x, gate, y, d_state_in=inplace, d_state_out=inplace, d_lengths=lengths,
                               d_workspace=buffers(s)[1])
    assert torch.equal(inplace, out) and torch.equal(y, apart)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64], ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_tensor_function_whatever_the_default_type(layout, default):
    """States and their gradients are float32 where torch makes other tensors by default."""
    x, gate, dy, state, dstate = values(16, "bfloat16", layout, 3, 150, 40)
    leaves = [v.detach().clone().requires_grad_() for v in (x, gate, state)]
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        y, last = thff.gated_scan(*leaves, layout=layout)
        torch.autograd.backward([y, last], [dy, dstate])
    finally:
        torch.set_default_dtype(before)
    assert last.dtype == torch.float32 and leaves[2].grad.dtype == torch.float32
    want = oracle.scan("bfloat16", layout, x, gate, state, None, dy, dstate)
    for name, v in (("y", y), ("state", last), ("dx", leaves[0].grad), ("dgate", leaves[1].grad),
                    ("dstate", leaves[2].grad)):
        oracle.check(name, v, want[name])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [0, 1, 40, 9000])
def test_saved_states_stay_in_their_bytes(layout, n):
    """Buffers cut from one block: nothing is written past saved_bytes(), which are none for n = 0."""
    batch, channels = 3, 37
    dims = (batch, n, channels) if layout == "channels_last" else (batch, channels, n)
    x, gate = torch.randn(dims).half().cuda(), torch.randn(dims).half().cuda()
    s = thff.ScanShape("half", batch, n, channels, layout=layout)
    size = s.saved_bytes()
    assert n > 0 or size == 0
    block = torch.full((64 + size + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    workspace, last = buffers(s)[1], torch.empty(batch, channels, device="cuda")
    thff.ThunderFFT_gated_scan(s, x, gate, torch.empty_like(x), d_state_out=last, d_saved=block[64:],
                               d_workspace=workspace)
    assert (block[:64] == 0x5A).all() and (block[64 + size:] == 0x5A).all()


@pytest.mark.parametrize("T", ["float", "bfloat16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [40, 700, 9000])
def test_huge_states_are_forgotten(T, layout, n):
    """States and gradients near the type's ends leave nothing behind closing gates, whose products
    are below any number: what follows has the size of small inputs.  (Each gate is 2e-9, so that
    the product of up to 4 is a normal number and that of more than 5 rounds to zero.)"""
    batch, channels = 2, 37
    x, gate, dy, state, dstate = values(17, T, layout, batch, n, channels)
    x, gate, dy = x.mul_(2.0 ** -30), gate.fill_(-20.0), dy.mul_(2.0 ** -30)
    state, dstate = state.sign() * 1e38, dstate.sign() * 1e38
    axis = 1 if layout == "channels_last" else 2
    x.narrow(axis, n // 2, 1).fill_(1e38)
    compare(T, layout, x, gate, dy, state, dstate)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_same_bits_whatever_the_workspace_held(layout):
    """Zeros, the chain's empty words, random words, plausible spans and what another call has left
    in the workspace change no bit, also while another stream keeps the card busy."""
    x, gate, dy, state, dstate = values(18, "half", layout, 2, 9000, 70)
    s = shape_of("half", layout, x, gate)
    saved, workspace = buffers(s)
    other = torch.empty_like(workspace)
    gen = torch.Generator(device="cuda").manual_seed(3)
    words = workspace.numel() // 8
    spans = torch.stack([torch.rand(words, device="cuda", generator=gen), torch.randn(words, device="cuda", generator=gen)], 1)
    contents = [torch.zeros_like(workspace), torch.full_like(workspace, 0xFF),
                torch.randint(0, 256, workspace.shape, dtype=torch.uint8, device="cuda", generator=gen),
                torch.cat([spans.flatten().view(torch.uint8), workspace.new_zeros(workspace.numel() - 8 * words)])]

    def calls(space, v):
        x, gate, dy, state, dstate = v
        y, dx, dg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        last, first = torch.empty_like(state), torch.empty_like(state)
        stream = torch.cuda.current_stream()
        thff.ThunderFFT_gated_scan_async(s, x, gate, y, d_state_in=state, d_state_out=last, d_saved=saved,
                                         d_workspace=space, stream=stream)
        kept = space.clone()
        thff.ThunderFFT_gated_scan_backward_async(s, dy, x, gate, saved, dx, dg, d_dstate_out=dstate, d_dstate_in=first,
                                                  d_workspace=space, stream=stream)
        return (y, last, dx, dg, first), kept

    ours = (x, gate, dy, state, dstate)
    want, _ = calls(workspace, ours)
    _, left = calls(other, values(19, "half", layout, 2, 9000, 70))  # another call's chains, complete
    a = torch.randn(2048, 2048, device="cuda", generator=gen)
    side = torch.cuda.Stream()
    for content in (*contents, left, other):
        for busy in (False, True):
            workspace.copy_(content)
            torch.cuda.synchronize()
            if busy:
                with torch.cuda.stream(side):
                    for _ in range(8):
                        a @ a
            got, _ = calls(workspace, ours)
            torch.cuda.synchronize()
            for v, w in zip(got, want):
                assert torch.equal(v, w)


# Shapes of more workgroups than one row of the grid has (2^21), with and without a chain:
# layout, batch, n, channels.
WIDE_GRIDS = [("channels_last", (1 << 21) + 5, 2, 1), ("channels_last", (1 << 20) + 3, 449, 1),
              ("channels_first", (1 << 20) + 7, 2, 128), ("channels_first", (1 << 13) + 1, 4097, 128)]


@pytest.mark.parametrize("shape", WIDE_GRIDS, ids=str)
def test_more_workgroups_than_a_row_of_the_grid(shape):
    """Gates of 0 (f = 1/2) and inputs of one value c a sequence: y[t] = c (1 - 2^-(t+1)), and with
    gradients of one value d, dx[t] = d (1 - 2^-(n-t)).  Sums of halves are exact in float as long as
    they differ from their limit, so each output is off by its rounding to half at most: 2^-11."""
    layout, batch, n, channels = shape
    first = layout == "channels_first"
    dims = (batch, channels, n) if first else (batch, n, channels)
    c = (torch.arange(batch, device="cuda") % 7 + 1).half().view(-1, 1, 1)
    d = (torch.arange(batch, device="cuda") % 5 + 1).half().view(-1, 1, 1)
    x, dy = c.expand(dims).contiguous(), d.expand(dims).contiguous()
    gate = torch.zeros_like(x)
    y, dx, dg = (torch.full_like(x, GUARD) for _ in range(3))
    last, dfirst = (torch.full((batch, channels), GUARD, device="cuda") for _ in range(2))
    s = thff.ScanShape("half", batch, n, channels, layout=layout)
    saved, workspace = buffers(s)
    print(layout, dims, flush=True)
    thff.ThunderFFT_gated_scan(s, x, gate, y, d_state_out=last, d_saved=saved, d_workspace=workspace)
    thff.ThunderFFT_gated_scan_backward(s, dy, x, gate, saved, dx, dg, d_dstate_in=dfirst, d_workspace=workspace)
    t = torch.arange(n, device="cuda", dtype=torch.float64).view((1, 1, n) if first else (1, n, 1))
    rising, falling = 1 - 0.5 ** (t + 1), 1 - 0.5 ** (n - t)
    step = max(1, (1 << 27) // (n * channels))
    for lo in range(0, batch, step):
        part = slice(lo, min(lo + step, batch))
        cs, ds = c[part].double(), d[part].double()
        for got, want in ((y, cs * rising), (dx, ds * falling)):
            assert bool(((got[part].double() - want).abs() <= want * 2.0 ** -11).all())
        # lam = 2 dx, h[t-1] - x = -c 2^-t: its own roundings are those of sums near c, 2^-24 of it.
        want = -0.5 * ds * falling * cs * 0.5 ** t
        bound = want.abs() * 2.0 ** -10 + ds * cs * 2.0 ** -23 + 2.0 ** -25
        assert bool(((dg[part].double() - want).abs() <= bound).all())
    cs, ds = c.double().view(-1, 1), d.double().view(-1, 1)
    assert bool(((last.double() - cs * (1 - 0.5 ** n)).abs() <= cs * 2.0 ** -23).all())
    assert bool(((dfirst.double() - ds * (1 - 0.5 ** n)).abs() <= ds * 2.0 ** -23).all())
