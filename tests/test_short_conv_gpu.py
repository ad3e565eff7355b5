"""The short causal convolution on the GPU against its definition in 64 bits: outputs, states and
gradients, in all types, for one token and for prompts."""
import pytest
import torch

import block_oracle as oracle
import thunderfft_amd as thff

pytestmark = pytest.mark.gpu
GUARD = -271.0


def values(seed, T, batch, n, channels, width):
    """x, weight, bias, state, dy, dstate on the GPU."""
    gen, dt = torch.Generator().manual_seed(seed), oracle.TYPES[T]

    def normal(*s):
        return torch.randn(*s, generator=gen)

    return (normal(batch, n, channels).to(dt).cuda(), (normal(channels, width) / 2).cuda(), (0.3 * normal(channels)).cuda(),
            normal(batch, width - 1, channels).to(dt).cuda(), normal(batch, n, channels).to(dt).cuda(),
            normal(batch, width - 1, channels).to(dt).cuda())


def placed(v, gap, offset):
    """A copy of v (batch, n, channels) with rows channels + gap apart, `offset` elements into its
    buffer, and whether what is around the rows is as it was."""
    batch, n, channels = v.shape
    stride = channels + gap
    whole = torch.full((offset + batch * n * stride + 64,), GUARD, dtype=v.dtype, device="cuda")
    out = whole[offset:offset + batch * n * stride].view(batch, n, stride)[..., :channels]
    out.copy_(v)

    def intact():
        around = whole.clone()
        around[offset:offset + batch * n * stride].view(batch, n, stride)[..., :channels] = GUARD
        return bool((around == GUARD).all())

    return out, intact


def run(T, x, weight, bias, state, dy, dstate, lengths=None, silu=True, gap=0, offset=0):
    batch, n, channels = x.shape
    width = weight.shape[1]
    print(f"{T} {batch} x {n} x {channels} width {width} silu {silu} gap {gap} offset {offset}", flush=True)
    nan = torch.full_like(x, float("nan"))
    (x, _), (dy, _), (y, y_ok), (dx, dx_ok) = (placed(v, gap, offset) for v in (x, dy, nan, nan))
    stride = channels + gap
    shape = thff.ConvShape(T, batch, n, channels, width, silu, x_stride=stride, y_stride=stride)
    last, first = (torch.full((batch * (width - 1) * channels + 8,), GUARD, dtype=x.dtype, device="cuda") for _ in range(2))
    thff.ThunderFFT_short_conv(shape, x, weight, bias, y, d_state_in=state, d_state_out=last, d_lengths=lengths)
    assert y_ok() and (last[-8:] == GUARD).all()
    workspace = torch.full((shape.workspace_bytes(),), 0xFF, dtype=torch.uint8, device="cuda")
    grads = torch.full((channels * (width + 1) + 8,), GUARD, device="cuda")
    dweight, dbias = grads[:channels * width].view(channels, width), grads[channels * width + 4:channels * (width + 1) + 4]
    thff.ThunderFFT_short_conv_backward(shape, dy, x, weight, bias, dx, dweight, dbias, d_state_in=state, d_dstate_out=dstate,
                                        d_dstate_in=first, d_lengths=lengths, d_workspace=workspace)
    assert dx_ok() and (first[-8:] == GUARD).all()
    assert (grads[channels * width:channels * width + 4] == GUARD).all() and (grads[-4:] == GUARD).all()
    rows = (batch, width - 1, channels)
    return dict(y=y, state=last[:-8].view(rows), dx=dx, dweight=dweight, dbias=dbias, dstate=first[:-8].view(rows))


def compare(T, x, weight, bias, state, dy, dstate, lengths=None, silu=True, **how):
    got = run(T, x, weight, bias, state, dy, dstate, lengths, silu, **how)
    want = oracle.conv(T, x, weight, bias, state, lengths, silu, dy, torch.zeros_like(state) if dstate is None else dstate)
    for name in want:
        oracle.check(name, got[name], want[name])


def ends(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(1, 1, 1), (2, 2, 3), (3, 3, 7), (2, 4, 8), (5, 16, 9), (2, 17, 64), (3, 33, 40), (1, 100, 130),
                                  (7, 31, 200), (2, 300, 24), (1, 1000, 5), (300, 3, 16), (1, 5, 2048)], ids=str)
def test_sizes(T, size):
    for width in (2, 3, 4):
        compare(T, *values(sum(size), T, *size, width))


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_without_activation_bias_and_states(T):
    x, weight, bias, state, dy, dstate = values(1, T, 3, 50, 72, 4)
    compare(T, x, weight, bias, state, dy, dstate, silu=False)
    compare(T, x, weight, None, state, dy, dstate)
    got = run(T, x, weight, bias, None, dy, None)
    want = oracle.conv(T, x, weight, bias, None, None, True, dy, torch.zeros_like(dstate))
    for name in want:
        oracle.check(name, got[name], want[name])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("how", [dict(gap=1), dict(gap=8), dict(offset=1), dict(offset=4), dict(gap=72, offset=8)], ids=str)
def test_strides_and_offsets(T, how):
    for size in ((3, 37, 72), (2, 20, 75), (2, 9, 3)):
        compare(T, *values(3, T, *size, 4), **how)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("width", [2, 3, 4])
def test_lengths(T, width):
    """Sequences that end early, before the first step, and outside [0, n]; junk behind the ends
    reaches nothing."""
    n = 45
    args = values(4, T, 9, n, 24, width)
    lengths = ends(0, 1, 2, 3, 16, 17, 44, n, 500)
    compare(T, *args, lengths=lengths)
    clean = run(T, *args, lengths=lengths)
    x, dy = args[0].clone(), args[4].clone()
    for b, end in enumerate(lengths.tolist()):
        x[b, end:] = float("nan")
        dy[b, end:] = float("inf")
    dirty = run(T, x, *args[1:4], dy, args[5], lengths=lengths)
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    below = run(T, *args, lengths=ends(-3, 1, 2, 3, 16, 17, 44, n, 500))
    assert torch.equal(below["y"], clean["y"]) and torch.equal(below["state"], clean["state"])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("channels", [3, 12, 40, 133])
def test_tokens_follow_prompts_in_a_pool(T, channels):
    """A prompt, a second chunk and single tokens, the states in place in rows of a pool, are as the
    whole sequence; rows of the pool that are no slot's stay, and empty places store nothing."""
    batch, n, width = 5, 60, 4
    x, weight, bias, *_ = values(5, T, batch, n, channels, width)
    whole = oracle.conv(T, x, weight, bias)
    pool = torch.full((9, width - 1, channels), GUARD, dtype=x.dtype, device="cuda")
    slots = ends(7, 0, -1, 3, 8)
    pool[slots[slots >= 0].long()] = 0
    kept = pool.clone()
    at, y = 0, torch.empty_like(x)
    for count in (33, 2, 18) + (1,) * 7:
        part = x[:, at:at + count].contiguous()
        shape = thff.ConvShape(T, batch, count, channels, width, states=9)
        out = torch.empty_like(part)
        thff.ThunderFFT_short_conv(shape, part, weight, bias, out, d_state_in=pool, d_state_out=pool, d_slots=slots)
        y[:, at:at + count] = out
        at += count
    value, bound = whole["y"]
    rows = [0, 1, 3, 4]
    oracle.check("y", y[rows], (value[rows], bound[rows]))
    assert torch.equal(pool[slots[rows].long()], x[rows, n - 3:])
    free = [r for r in range(9) if r not in (7, 0, 3, 8)]
    assert torch.equal(pool[free], kept[free])
    # The empty place had no past.
    last = oracle.conv(T, x[2:3, n - 1:], weight, bias)["y"]
    oracle.check("empty", y[2:3, n - 1:], last)
    # A slot behind the pool is none either.
    thff.ThunderFFT_short_conv(thff.ConvShape(T, 1, 1, channels, width, states=9), x[:1, :1].contiguous(), weight, bias, y[:1, :1],
                               d_state_in=pool, d_state_out=pool, d_slots=ends(9))
    assert torch.equal(pool[free], kept[free])


def test_no_steps_and_nothing():
    """No steps copy the states and their gradients; no sequences leave the weights' gradients zero."""
    for width in (2, 4):
        x, weight, bias, state, dy, dstate = values(6, "half", 3, 0, 21, width)
        got = run("half", x, weight, bias, state, dy, dstate)
        assert torch.equal(got["state"], state) and torch.equal(got["dstate"], dstate)
        assert (got["dweight"] == 0).all() and (got["dbias"] == 0).all()
    shape = thff.ConvShape("half", 0, 9, 21, 4)
    dweight, dbias = torch.full((21, 4), GUARD, device="cuda"), torch.full((21,), GUARD, device="cuda")
    thff.ThunderFFT_short_conv_backward(shape, 0, 0, 0, 0, 0, dweight, dbias)
    assert (dweight == 0).all() and (dbias == 0).all()


@pytest.mark.parametrize("cols", [16, 21])
def test_gradients_wanted_singly(cols):
    x, weight, bias, state, dy, dstate = values(7, "half", 6, 90, cols, 3)
    both = run("half", x, weight, bias, state, dy, dstate)
    shape = thff.ConvShape("half", 6, 90, cols, 3)
    for w, b in ((True, False), (False, True), (False, False)):
        dw, db, dx = torch.empty_like(weight), torch.empty_like(bias), torch.zeros_like(x)
        work = torch.empty(shape.workspace_bytes(), dtype=torch.uint8, device="cuda") if w or b else None
        thff.ThunderFFT_short_conv_backward(shape, dy, x, weight, bias, dx, dw if w else None, db if b else None, d_state_in=state,
                                            d_dstate_out=dstate, d_workspace=work)
        assert torch.equal(dx, both["dx"])
        assert not w or torch.equal(dw, both["dweight"])
        assert not b or torch.equal(db, both["dbias"])


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_non_finite_values_stay_near(junk):
    """A NaN or an infinity reaches the outputs of its channel and the width - 1 steps behind it."""
    x, weight, bias, *_ = values(8, "half", 2, 70, 24, 4)
    shape = thff.ConvShape("half", 2, 70, 24, 4)
    y, z = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_short_conv(shape, x, weight, bias, y)
    x[1, 33, 5] = junk
    thff.ThunderFFT_short_conv(shape, x, weight, bias, z)
    reached = torch.zeros_like(x, dtype=torch.bool)
    reached[1, 33:37, 5] = True
    assert torch.equal(y[~reached], z[~reached])
    assert (z[1, 33:37, 5].isnan() | z[1, 33:37, 5].isinf() | (z[1, 33:37, 5] == 0)).all()


def test_large_sums_are_closed_and_open():
    """silu far from zero: 0 on one side, the value on the other, no NaN."""
    x = torch.tensor([[[-3e4], [-200.0], [-90.0], [90.0], [3e4]]], device="cuda")
    weight, y = torch.tensor([[0.0, 1.0]], device="cuda"), torch.empty_like(x)
    thff.ThunderFFT_short_conv(thff.ConvShape("float", 1, 5, 1, 2), x, weight, None, y)
    assert torch.equal(y.flatten()[:2], torch.zeros(2, device="cuda")) and float(y[0, 2].abs()) < 1e-36
    assert torch.equal(y[0, 3:], x[0, 3:])


@pytest.mark.parametrize("size", [(3, 200, 264), (2, 4000, 16)], ids=str)
def test_same_bits_each_time(size):
    args = values(9, "bfloat16", *size, 4)
    first = run("bfloat16", *args)
    for _ in range(3):
        again = run("bfloat16", *args)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_streams_and_graph_replays():
    """On a stream of its own, captured, and replayed with new inputs and eager calls between."""
    args = values(10, "bfloat16", 4, 300, 136, 4)
    x, weight, bias, state, dy, dstate = args
    shape = thff.ConvShape("bfloat16", 4, 300, 136, 4)
    y, dx, last, first = torch.empty_like(x), torch.empty_like(x), torch.empty_like(state), torch.empty_like(state)
    dw, db = torch.empty_like(weight), torch.empty_like(bias)
    workspace = torch.empty(shape.workspace_bytes(), dtype=torch.uint8, device="cuda")

    def calls(stream):
        thff.ThunderFFT_short_conv_async(shape, x, weight, bias, y, d_state_in=state, d_state_out=last, stream=stream)
        thff.ThunderFFT_short_conv_backward_async(shape, dy, x, weight, bias, dx, dw, db, d_state_in=state, d_dstate_out=dstate,
                                                  d_dstate_in=first, d_workspace=workspace, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls(side)
    torch.cuda.synchronize()
    got = dict(y=y, state=last, dx=dx, dweight=dw, dbias=db, dstate=first)
    want = run("bfloat16", *args)
    assert all(torch.equal(want[name], v) for name, v in got.items())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for k in range(4):
        new = values(50 + k, "bfloat16", 4, 300, 136, 4)
        for old, v in zip(args, new):
            old.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = run("bfloat16", *new)
        for name, v in got.items():
            assert torch.equal(want[name], v), (k, name)


@pytest.mark.parametrize("fused", [False, True])
def test_tensor_function(fused):
    """short_conv's outputs and gradients, x dense or the half of a projection's rows."""
    x, weight, bias, state, dy, dstate = values(11, "bfloat16", 3, 40, 64, 4)
    lengths = ends(40, 7, 0)
    if fused:
        x = torch.cat([x, torch.full_like(x, float("nan"))], 2)[..., :64]
    leaves = [v.detach().requires_grad_() for v in (x, weight, bias, state)]
    y, last = thff.short_conv(*leaves, lengths)
    torch.autograd.backward([y, last], [dy, dstate])
    want = oracle.conv("bfloat16", x, weight, bias, state, lengths, True, dy, dstate)
    got = dict(zip(("dx", "dweight", "dbias", "dstate"), (v.grad for v in leaves)), y=y, state=last)
    for name in want:
        oracle.check(name, got[name], want[name])
    # The last state alone, and without one.
    y, last = thff.short_conv(*leaves[:2])
    last.sum().backward()
    y, last = thff.short_conv(leaves[0], weight, silu=False)
    y.sum().backward()
    with torch.no_grad():
        y, _ = thff.short_conv(x, weight, None, None, None, False)
    oracle.check("y", y, oracle.conv("bfloat16", x, weight, None, silu=False)["y"])
    with pytest.raises(ValueError, match="state must have shape"):
        thff.short_conv(x, weight, bias, state[:, :2])
    with pytest.raises(ValueError, match="width 2 to 4"):
        thff.short_conv(x, torch.zeros(64, 5, device="cuda"))


@pytest.mark.parametrize("T,width", [("half", 2), ("bfloat16", 3), ("float", 4)])
def test_many_values(T, width):
    """Past 2^25 values a lane has other channels: a few of them, the first and the last, against the
    formulas in 64 bits, as no channel depends on another."""
    v = values(11, T, 3, 5600, 2051, width)
    lengths = ends(5600, 17, 5589)
    got = run(T, *v, lengths=lengths, gap=5)
    few = torch.tensor([0, 1, 2, 3, 1023, 2044, 2047, 2048, 2049, 2050], device="cuda")
    x, weight, bias, state, dy, dstate = (t.index_select(0 if t.dim() < 3 else 2, few) for t in v)
    want = oracle.conv(T, x, weight, bias, state, lengths, True, dy, dstate)
    for name in want:
        part = got[name].index_select(0 if name in ("dweight", "dbias") else 2, few)
        oracle.check(name, part, want[name])


def test_offsets_past_32_bits():
    """Rows further than 2^32 bytes into the buffer: the last channels of a long sequence of one
    width as those of a short one."""
    n, channels = (1 << 31) // 1024 + 300, 1024
    x = torch.empty(1, n, channels, dtype=torch.float16, device="cuda").normal_()
    weight = torch.randn(channels, 4, device="cuda")
    y = torch.empty_like(x)
    thff.ThunderFFT_short_conv(thff.ConvShape("half", 1, n, channels, 4), x, weight, None, y)
    tail = x[:, -100:].contiguous()
    z, state = torch.empty_like(tail), x[:, -103:-100].contiguous()
    thff.ThunderFFT_short_conv(thff.ConvShape("half", 1, 100, channels, 4), tail, weight, None, z, d_state_in=state)
    assert torch.equal(y[:, -100:], z)
    dx, dz = torch.empty_like(x), torch.empty_like(tail)
    shape = thff.ConvShape("half", 1, n, channels, 4)
    thff.ThunderFFT_short_conv_backward(shape, y, x, weight, None, dx)
    thff.ThunderFFT_short_conv_backward(thff.ConvShape("half", 1, 100, channels, 4), z, tail, weight, None, dz, d_state_in=state)
    assert torch.equal(dx[:, -100:], dz)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("silu", [True, False])
def test_same_bits_however_a_sequence_is_cut(T, silu):
    """A sequence in one call, and in calls of other lengths that hand the state on, fall otherwise into the
    kernels' tiles: outputs, states and gradients of values have the same bits."""
    n, channels, width = 1500, 1024, 4
    x, weight, bias, _, dy, _ = values(41, T, 1, n, channels, width)
    whole = thff.ConvShape(T, 1, n, channels, width, silu)
    y, dx, last = torch.empty_like(x), torch.empty_like(x), x.new_empty(1, width - 1, channels)
    thff.ThunderFFT_short_conv(whole, x, weight, bias, y, d_state_out=last)
    thff.ThunderFFT_short_conv_backward(whole, dy, x, weight, bias, dx)
    for count in (1, 7, 24, 401):
        state, z = torch.zeros_like(last), torch.empty_like(x)
        for at in range(0, n, count):
            now = min(count, n - at)
            part = thff.ConvShape(T, 1, now, channels, width, silu)
            thff.ThunderFFT_short_conv_async(part, x[:, at:], weight, bias, z[:, at:], d_state_in=state, d_state_out=state)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(last, state), count
    # The gradients of all but the last steps of a call, which others behind it reach too.
    for at in range(1, 40, 3):
        part, dz = thff.ConvShape(T, 1, n - at, channels, width, silu), torch.empty_like(x[:, at:])
        thff.ThunderFFT_short_conv_backward(part, dy[:, at:], x[:, at:], weight, bias, dz, d_state_in=x[:, at - 3:at].contiguous()
                                            if at >= 3 else torch.cat([torch.zeros_like(x[:, at:3]), x[:, :at]], 1))
        assert torch.equal(dz, dx[:, at:]), at
