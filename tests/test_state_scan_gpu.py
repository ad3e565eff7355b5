"""The state space scan on the GPU against its definition in 64 bits: outputs, states and gradients,
in all types, orders and groups, for one token, for prompts and for long sequences in segments."""
import math

import pytest
import torch

import block_oracle as oracle
import thunderfft_amd as thff

pytestmark = pytest.mark.gpu
GUARD = -271.0
SHARED = ("b", "c")
VALUES = ("x", "delta", "gate")


def values(seed, T, batch, n, channels, order, groups=1):
    """The arguments by name, on the GPU: steps from a thousandth to a tenth, rates from one up."""
    gen, dt = torch.Generator().manual_seed(seed), oracle.TYPES[T]

    def normal(*s):
        return torch.randn(*s, generator=gen)

    v = dict(x=normal(batch, n, channels).to(dt), delta=(0.5 * normal(batch, n, channels)).to(dt),
             a=-(torch.arange(1, order + 1) * (0.2 * normal(channels, order)).exp()), b=normal(batch, n, groups, order).to(dt),
             c=normal(batch, n, groups, order).to(dt), skip=1 + 0.2 * normal(channels), gate=normal(batch, n, channels).to(dt),
             delta_bias=torch.linspace(-7, -2, channels), state=normal(batch, channels, order))
    return {k: t.cuda() for k, t in v.items()} | dict(dy=normal(batch, n, channels).to(dt).cuda(),
                                                      dstate=normal(batch, channels, order).cuda())


def ends(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def placed(v, gap, offset):
    """A copy of v (batch, n, ...) with rows `gap` more apart than they are long, `offset` elements
    into its buffer, and whether what is around the rows is as it was."""
    flat = v.flatten(2)
    batch, n, row = flat.shape
    stride = row + gap
    whole = torch.full((offset + batch * n * stride + 64,), GUARD, dtype=v.dtype, device="cuda")
    out = whole[offset:offset + batch * n * stride].view(batch, n, stride)[..., :row]
    out.copy_(flat)

    def intact():
        around = whole.clone()
        around[offset:offset + batch * n * stride].view(batch, n, stride)[..., :row] = GUARD
        return bool((around == GUARD).all())

    return out, intact


def run(T, v, lengths=None, gap=0, offset=0):
    """Outputs and gradients by the calls on device buffers; every buffer is guarded."""
    batch, n, channels = v["x"].shape
    groups, order = v["b"].shape[2:]
    row = groups * order
    print(f"{T} {batch} x {n} x {channels} order {order} groups {groups} gap {gap} offset {offset} "
          f"without {[k for k in v if v[k] is None]}", flush=True)
    stride = channels + gap
    shape = thff.StateShape(T, batch, n, channels, order, groups, stride, stride, stride, row + gap, row + gap, stride)
    at = {k: placed(v[k], gap, offset)[0] for k in ("x", "delta", "b", "c", "dy")}
    gate = None if v["gate"] is None else placed(v["gate"], gap, offset)[0]
    nan = torch.full_like(v["x"], float("nan"))
    out = {k: placed(nan, gap, offset) for k in ("y", "dx", "ddelta", "dgate")}
    out |= {k: placed(torch.full_like(v["b"], float("nan")), gap, offset) for k in ("db", "dc")}
    sizes = dict(state=batch * channels * order, dstate=batch * channels * order, da=channels * order, dskip=channels,
                 ddelta_bias=channels)
    weights = {k: torch.full((size + 4,), GUARD, device="cuda") for k, size in sizes.items()}

    def scratch(count):
        return torch.full((count + 64,), 0xFF, dtype=torch.uint8, device="cuda")

    saved, workspace = scratch(shape.saved_bytes()), scratch(shape.forward_bytes())
    thff.ThunderFFT_state_scan(shape, at["x"], at["delta"], v["a"], at["b"], at["c"], out["y"][0], d_skip=v["skip"], d_gate=gate,
                               d_delta_bias=v["delta_bias"], d_state_in=v["state"], d_state_out=weights["state"], d_lengths=lengths,
                               d_saved=saved, d_workspace=workspace)
    assert (workspace[-64:] == 0xFF).all()
    assert (saved[-64:] == 0xFF).all()
    workspace = scratch(shape.workspace_bytes())
    thff.ThunderFFT_state_scan_backward(
        shape, at["dy"], at["x"], at["delta"], v["a"], at["b"], at["c"], saved, out["dx"][0], out["ddelta"][0], weights["da"],
        out["db"][0], out["dc"][0], d_skip=v["skip"], d_dskip=weights["dskip"], d_gate=gate,
        d_dgate=None if gate is None else out["dgate"][0], d_delta_bias=v["delta_bias"], d_ddelta_bias=weights["ddelta_bias"],
        d_dstate_out=v["dstate"], d_dstate_in=weights["dstate"], d_lengths=lengths, d_workspace=workspace)
    assert (workspace[-64:] == 0xFF).all()
    got = {}
    for k, (t, intact) in out.items():
        assert intact(), k
        got[k] = t.reshape(v["b"].shape) if k in ("db", "dc") else t
    for k, t in weights.items():
        assert (t[sizes[k]:] == GUARD).all(), k
        got[k] = t[:sizes[k]].view(channels, order) if k == "da" else t[:sizes[k]].view(
            (batch, channels, order) if k in ("state", "dstate") else (channels,))
    if gate is None:
        del got["dgate"]
    return got


def wanted(T, v, lengths=None):
    return oracle.state(T, v["x"], v["delta"], v["a"], v["b"], v["c"], v["skip"], v["gate"], v["delta_bias"], v["state"], lengths,
                        v["dy"], v["dstate"])


def compare(T, v, lengths=None, **how):
    got, want = run(T, v, lengths, **how), wanted(T, v, lengths)
    assert got.keys() == want.keys()
    for name in want:
        oracle.check(name, got[name], want[name])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (2, 2, 3, 4), (3, 3, 17, 5), (2, 15, 8, 8), (1, 16, 64, 16), (2, 17, 65, 16),
                                  (3, 31, 40, 12), (1, 33, 130, 3), (2, 64, 16, 16), (1, 100, 33, 24), (2, 50, 20, 32), (1, 70, 9, 33),
                                  (2, 40, 12, 64), (40, 5, 48, 16), (130, 45, 24, 16), (140, 70, 9, 12),
                                  (300, 20, 17, 16)], ids=str)
def test_sizes(T, size):
    compare(T, values(sum(size), T, *size))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(2, 40, 12, 7, 12), (1, 20, 96, 16, 2), (3, 9, 300, 16, 3), (2, 35, 8, 40, 4)], ids=str)
def test_groups(T, size):
    compare(T, values(1, T, *size))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("without", [("gate",), ("skip",), ("delta_bias",), ("state",), ("dstate",),
                                     ("gate", "skip", "delta_bias", "state", "dstate")], ids=str)
def test_optional_arguments(T, without):
    v = values(2, T, 3, 37, 24, 16)
    if "delta_bias" in without:
        v["delta"] -= 3
    compare(T, v | {k: None for k in without})


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("how", [dict(gap=1), dict(gap=8), dict(offset=1), dict(offset=4), dict(gap=48, offset=8)], ids=str)
def test_strides_and_offsets(T, how):
    for size in ((3, 37, 72, 16, 1), (2, 20, 30, 5, 2)):
        compare(T, values(3, T, *size), **how)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("order", [4, 16, 24])
def test_lengths(T, order):
    """Sequences that end early, before the first step, and outside [0, n]; junk behind the ends
    reaches nothing."""
    n = 75
    v = values(4, T, 9, n, 24, order)
    lengths = ends(0, 1, 15, 16, 17, 32, 64, n, 500)
    compare(T, v, lengths)
    clean = run(T, v, lengths)
    dirty = {k: t.clone() for k, t in v.items()}
    for b, end in enumerate(lengths.tolist()):
        for name, junk in (("x", "nan"), ("delta", "inf"), ("gate", "-inf"), ("b", "inf"), ("c", "nan"), ("dy", "nan")):
            dirty[name][b, end:] = float(junk)
    got = run(T, dirty, lengths)
    for name in clean:
        assert torch.equal(clean[name], got[name]), name
    below = run(T, v, ends(-3, 1, 15, 16, 17, 32, 64, n, 500))
    for name in clean:
        assert torch.equal(clean[name], below[name]), name


@pytest.mark.parametrize("n", [1, 2, 5, 15, 34])
@pytest.mark.parametrize("channels,order", [(64, 16), (70, 3), (40, 40)])
def test_a_few_steps_of_all_lengths(n, channels, order):
    """Sequences of 0 to n steps: what lies behind each length is 0, wherever it falls in a block."""
    v = values(27 + n, "half", n + 1, n, channels, order)
    compare("half", v, ends(*range(n, -1, -1)))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(1, 3000, 20, 16, 1), (2, 1500, 6, 5, 2), (1, 2500, 70, 4, 1), (1, 1100, 9, 40, 1)], ids=str)
def test_long_sequences(T, size):
    compare(T, values(5, T, *size))


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_long_sequences_that_end_early(T):
    v = values(6, T, 4, 2100, 24, 16)
    compare(T, v, ends(2100, 1000, 5, 0))


def test_many_sequences_that_end_early():
    """As many waves as have 8 lanes a channel."""
    v = values(19, "half", 150, 100, 40, 16)
    compare("half", v, (torch.arange(150, device="cuda") * 37 % 101).to(torch.int32))


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_steps_of_all_sizes(T):
    """Steps from nothing, which keep the states, to ones that leave nothing of them; rates of zero."""
    v = values(7, T, 2, 60, 32, 16)
    v["delta"][0, ::3] = -40
    v["delta"][0, 1::3] = 40
    v["delta"][1] = 6
    v["a"][:, 3] = 0
    v["a"][5] = -30
    compare(T, v)


def test_growing_states():
    """Positive rates: the states grow."""
    v = values(8, "float", 2, 40, 16, 8)
    v["a"] = -0.3 * v["a"]
    compare("float", v)


@pytest.mark.parametrize("order", [4, 16, 40])
def test_states_of_zero_do_not_grow(order):
    """A positive rate and long steps: the factor of some hundred steps is out of range, the states that it
    would take there are zero.  Only the last steps have an x, only the first ones a dy."""
    n, few = 2000, 5
    v = values(17, "float", 1, n, 24, order)
    v["a"] = v["a"].abs() * 0.0 + 0.5
    v["delta"][:] = 6
    v["state"] = v["dstate"] = None
    v["x"][:, :-few] = 0
    v["dy"][:, few:] = 0
    got = run("float", v)
    last = run("float", dict(v, **{k: v[k][:, -few:].contiguous() for k in ("x", "delta", "b", "c", "gate", "dy")}))
    first = run("float", dict(v, **{k: v[k][:, :few].contiguous() for k in ("x", "delta", "b", "c", "gate", "dy")}))
    assert (got["y"][:, :-few] == 0).all() and (got["dx"][:, few:] == 0).all()
    for name, want in (("y", last["y"]), ("state", last["state"])):
        # The same steps in fp32, whose dt and factors the two runs round alike.
        assert torch.allclose(got[name][:, -few:] if name == "y" else got[name], want, rtol=2.0 ** -20, atol=0), name
    assert torch.allclose(got["dx"][:, :few], first["dx"], rtol=2.0 ** -18, atol=2.0 ** -18 * first["dx"].abs().max().item())


@pytest.mark.parametrize("order", [4, 16, 40])
@pytest.mark.parametrize("power", [250, 257, 260])
def test_small_states_that_grow(order, power):
    """A state of 2^-140 that 96 steps in the middle take up by 2^power: the factor alone is out of range,
    its product with the state is not.  The steps beside them have a dt of 0; the gradient of the state goes
    back alike.  (dt a) is off by 2^-20 of `power` at most, the state at first by 2^-150 of 2^-140 a step, which
    a step's growth by 2^2.6 and more makes 2^-9.6 of it in all: 2^-8."""
    n, at, few = 2000, 960, 96
    v = values(25, "float", 1, n, 24, order)
    v["a"] = torch.full_like(v["a"], 0.5)
    dt = power * math.log(2.0) / few / 0.5
    v["delta"][:] = -200
    v["delta"][:, at:at + few] = math.log(math.expm1(dt))
    v |= dict(delta_bias=None, gate=None, skip=None)
    for name in ("x", "dy"):
        v[name][:] = 0
    small, nothing = torch.full_like(v["state"], 2.0 ** -140), torch.zeros_like(v["state"])
    # delta is rounded to fp32, with dt = softplus(delta) by the slope of it, 1 at most.
    slack = few * 0.5 * 4 * 2.0 ** -24 / math.log(2.0)
    assert slack < 2.0 ** -10
    for given, name in ((dict(state=small, dstate=nothing), "state"), (dict(state=nothing, dstate=small), "dstate")):
        got = run("float", v | given)
        end = got[name].double() / 2.0 ** (power - 140)
        assert ((end - 1).abs() < 2.0 ** -8).all(), (name, end.min().item(), end.max().item())
        if name == "state":
            assert torch.isfinite(got["y"]).all()


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(37, 5), (24, 16), (9, 64), (16, 24)], ids=str)
def test_tokens_follow_prompts_in_a_pool(T, size):
    """A prompt, a second chunk and single tokens, the states in place in rows of a pool, are as the
    whole sequence; rows of the pool that are no slot's stay, and empty places store nothing."""
    channels, order = size
    batch, n = 5, 60
    v = values(9, T, batch, n, channels, order)
    v["state"] = None
    whole = oracle.state(T, v["x"], v["delta"], v["a"], v["b"], v["c"], v["skip"], v["gate"], v["delta_bias"])
    pool = torch.full((9, channels, order), GUARD, device="cuda")
    slots, rows = ends(7, 0, -1, 3, 8), [0, 1, 3, 4]
    pool[slots[rows].long()] = 0
    kept = pool.clone()
    at, y = 0, torch.empty_like(v["x"])
    for count in (33, 2, 18) + (1,) * 7:
        part = {k: v[k][:, at:at + count].contiguous() for k in VALUES + SHARED}
        shape = thff.StateShape(T, batch, count, channels, order, states=9)
        out = torch.empty_like(part["x"])
        work = torch.empty(shape.forward_bytes(), dtype=torch.uint8, device="cuda")
        thff.ThunderFFT_state_scan(shape, part["x"], part["delta"], v["a"], part["b"], part["c"], out, d_skip=v["skip"],
                                   d_gate=part["gate"], d_delta_bias=v["delta_bias"], d_state_in=pool, d_state_out=pool,
                                   d_slots=slots, d_workspace=work)
        y[:, at:at + count] = out
        at += count
    for name, got in (("y", y), ("state", pool[slots.long()])):
        value, bound = whole[name]
        oracle.check(name, got[rows], (value[rows], bound[rows]))
    free = [r for r in range(9) if r not in (7, 0, 3, 8)]
    assert torch.equal(pool[free], kept[free])
    # The empty place had no past.
    last = {k: v[k][2:3, n - 1:] for k in VALUES + SHARED}
    want = oracle.state(T, last["x"], last["delta"], v["a"], last["b"], last["c"], v["skip"], last["gate"], v["delta_bias"])
    oracle.check("empty", y[2:3, n - 1:], want["y"])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(70, 16, 1, 1), (3, 24, 3, 3), (260, 48, 16, 2), (4, 40, 33, 1), (5, 1000, 16, 1)], ids=str)
def test_one_token(T, size):
    """n = 1, with lengths of 0 and 1, a shape of strides, and without each optional argument."""
    batch, channels, order, groups = size
    v = values(10, T, batch, 1, channels, order, groups)
    lengths = (torch.arange(batch, device="cuda") % 3 != 1).to(torch.int32)
    for without in ((), ("gate",), ("skip", "state"), ("delta_bias",)):
        w = v | {k: None for k in without}
        for end in (None, lengths):
            want = oracle.state(T, w["x"], w["delta"], w["a"], w["b"], w["c"], w["skip"], w["gate"], w["delta_bias"], w["state"], end)
            at = {k: None if w[k] is None else placed(w[k], 3, 1)[0] for k in VALUES + SHARED}
            y, intact = placed(torch.full_like(v["x"], float("nan")), 3, 1)
            row = groups * order + 3
            shape = thff.StateShape(T, batch, 1, channels, order, groups, *(channels + 3,) * 3, row, row, channels + 3)
            state = torch.full((batch * channels * order + 4,), GUARD, device="cuda")
            work = torch.empty(shape.forward_bytes(), dtype=torch.uint8, device="cuda")
            thff.ThunderFFT_state_scan(shape, at["x"], at["delta"], w["a"], at["b"], at["c"], y, d_skip=w["skip"], d_gate=at["gate"],
                                       d_delta_bias=w["delta_bias"], d_state_in=w["state"], d_state_out=state, d_lengths=end,
                                       d_workspace=work)
            assert intact() and (state[-4:] == GUARD).all()
            oracle.check("y", y, want["y"])
            oracle.check("state", state[:-4].view(batch, channels, order), want["state"])


def test_no_steps_and_nothing():
    """No steps copy the states and their gradients; no sequences leave the weights' gradients zero."""
    for order in (5, 16):
        v = values(11, "half", 3, 0, 21, order)
        got = run("half", v)
        assert torch.equal(got["state"], v["state"]) and torch.equal(got["dstate"], v["dstate"])
        assert all((got[k] == 0).all() for k in ("da", "dskip", "ddelta_bias"))
    shape = thff.StateShape("half", 0, 9, 21, 5)
    da, dskip, dbias = (torch.full(s, GUARD, device="cuda") for s in ((21, 5), (21,), (21,)))
    thff.ThunderFFT_state_scan_backward(shape, 0, 0, 0, 0, 0, 0, 0, 0, 0, da, 0, 0, d_dskip=dskip, d_ddelta_bias=dbias)
    assert all((t == 0).all() for t in (da, dskip, dbias))


@pytest.mark.parametrize("name,junk", [("x", "nan"), ("x", "inf"), ("delta", "nan"), ("b", "nan"), ("c", "inf"), ("gate", "nan")])
def test_non_finite_values_stay_where_they_belong(name, junk):
    """Outputs that do not depend on a NaN or an infinity are as without it; those of its step that do are not finite."""
    v = values(12, "half", 2, 700, 24, 16, 2)
    clean = run("half", v)
    w = {k: t.clone() for k, t in v.items()}
    if name in SHARED:
        w[name][1, 333, 1, 4] = float(junk)
    else:
        w[name][1, 333, 17] = float(junk)
    got = run("half", w)
    touched = torch.zeros_like(v["x"], dtype=torch.bool)
    if name in SHARED:
        touched[1, 333:334 if name == "c" else 700, 12:] = True
    else:
        touched[1, 333:334 if name == "gate" else 700, 17] = True
    assert torch.equal(got["y"][~touched], clean["y"][~touched])
    assert not torch.isfinite(got["y"][1, 333][touched[1, 333]]).any()


@pytest.mark.parametrize("size", [(3, 200, 72, 16), (1, 3000, 24, 16), (2, 100, 20, 40)], ids=str)
def test_same_bits_each_time(size):
    v = values(13, "bfloat16", *size)
    first = run("bfloat16", v)
    for _ in range(3):
        again = run("bfloat16", v)
        for name in first:
            assert torch.equal(first[name], again[name]), name


@pytest.mark.parametrize("size", [(4, 100, 136, 16), (1, 3000, 24, 16)], ids=str)
def test_streams_and_graph_replays(size):
    """On a stream of its own, captured, and replayed with new inputs and eager calls between."""
    v = values(14, "bfloat16", *size)
    batch, n, channels, order = size
    shape = thff.StateShape("bfloat16", *size)
    out = {k: torch.empty_like(v[k[1:]]) for k in ("dx", "ddelta", "dgate", "da", "db", "dc", "dskip", "ddelta_bias", "dstate")}
    out |= dict(y=torch.empty_like(v["x"]), state=torch.empty_like(v["state"]))
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    workspace = torch.empty(shape.workspace_bytes(), dtype=torch.uint8, device="cuda")

    def calls(stream):
        thff.ThunderFFT_state_scan_async(shape, v["x"], v["delta"], v["a"], v["b"], v["c"], out["y"], d_skip=v["skip"],
                                         d_gate=v["gate"], d_delta_bias=v["delta_bias"], d_state_in=v["state"],
                                         d_state_out=out["state"], d_saved=saved, d_workspace=workspace, stream=stream)
        thff.ThunderFFT_state_scan_backward_async(
            shape, v["dy"], v["x"], v["delta"], v["a"], v["b"], v["c"], saved, out["dx"], out["ddelta"], out["da"], out["db"],
            out["dc"], d_skip=v["skip"], d_dskip=out["dskip"], d_gate=v["gate"], d_dgate=out["dgate"], d_delta_bias=v["delta_bias"],
            d_ddelta_bias=out["ddelta_bias"], d_dstate_out=v["dstate"], d_dstate_in=out["dstate"], d_workspace=workspace,
            stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls(side)
    torch.cuda.synchronize()
    want = run("bfloat16", v)
    assert all(torch.equal(want[name], t) for name, t in out.items())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for k in range(4):
        new = values(50 + k, "bfloat16", *size)
        for name in v:
            v[name].copy_(new[name])
        graph.replay()
        torch.cuda.synchronize()
        want = run("bfloat16", new)
        for name, t in out.items():
            assert torch.equal(want[name], t), (k, name)


@pytest.mark.parametrize("fused", [False, True])
def test_tensor_function(fused):
    """state_scan's outputs and gradients, from dense arguments and from slices of projections' rows."""
    v = values(15, "bfloat16", 3, 40, 64, 16, 2)
    lengths = ends(40, 7, 0)
    if fused:
        v["gate"] = torch.cat([torch.full_like(v["x"], float("nan")), v["gate"]], 2)[..., 64:]
        rows = torch.cat([torch.zeros_like(v["x"][..., :5]), v["b"].flatten(2), v["c"].flatten(2)], 2)
        v["b"], v["c"] = rows[..., 5:37].unflatten(2, (2, 16)), rows[..., 37:].unflatten(2, (2, 16))
    names = ("x", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "state")
    leaves = [v[k].detach().requires_grad_() for k in names]
    y, last = thff.state_scan(*leaves, lengths)
    torch.autograd.backward([y, last], [v["dy"], v["dstate"]])
    want = wanted("bfloat16", v, lengths)
    got = {"d" + k: t.grad for k, t in zip(names, leaves)} | dict(y=y, state=last)
    for name in want:
        oracle.check(name, got[name], want[name])
    # One group without an axis of its own, no optional arguments, gradients of some alone.
    w = values(16, "float", 2, 30, 20, 8)
    x, a = w["x"].requires_grad_(), w["a"].requires_grad_()
    y, last = thff.state_scan(x, w["delta"], a, w["b"][:, :, 0], w["c"][:, :, 0])
    last.backward(w["dstate"])
    w |= dict(skip=None, gate=None, delta_bias=None, state=None, dy=torch.zeros_like(w["dy"]))
    want = wanted("float", w)
    for name, t in (("y", y), ("state", last), ("dx", x.grad), ("da", a.grad)):
        oracle.check(name, t, want[name])
    with pytest.raises(ValueError, match="groups must divide"):
        thff.state_scan(w["x"], w["delta"], w["a"], w["b"].expand(-1, -1, 3, -1), w["c"].expand(-1, -1, 3, -1))
    with pytest.raises(ValueError, match="order 1 to 64"):
        thff.state_scan(w["x"], w["delta"], torch.zeros(20, 65, device="cuda"), w["b"], w["c"])


def test_gradients_against_differences():
    """Along a random direction of all arguments at once: float32 outputs are off by some 1e-6 of sums
    of order ten, and a step of 2^-6 of smooth functions by its square."""
    v = values(17, "float", 2, 23, 12, 6)
    names = ("x", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "state")
    gen = torch.Generator().manual_seed(18)
    way = {k: 0.1 * torch.randn(v[k].shape, generator=gen).cuda() for k in names}

    def outputs(step):
        y, last = thff.state_scan(*(v[k] + step * way[k] for k in names))
        return float((y.double() * v["dy"]).sum() + (last.double() * v["dstate"]).sum())

    got = run("float", v)
    along = sum(float((got["d" + k].double() * way[k].double()).sum()) for k in names)
    quotient = (outputs(2.0 ** -6) - outputs(-(2.0 ** -6))) * 2 ** 5
    assert abs(quotient - along) < 2e-3 * max(1.0, abs(along)), (quotient, along)


@pytest.mark.parametrize("n", [300, 1])
def test_offsets_past_32_bits(n):
    """Rows 2^22 apart, the last ones more than 2^32 bytes into their buffers: the same bits as of dense rows."""
    rows, stride, channels, order = 600, 1 << 22, 40, 16
    v = values(31, "half", rows // n, n, channels, order)
    names = dict(x=0, delta=64, gate=128, b=192, c=256, dy=320)
    far = torch.empty(rows, stride, dtype=torch.float16, device="cuda")
    out = torch.empty_like(far)
    for name, at in names.items():
        part = v[name].reshape(rows, -1)
        far[:, at:at + part.shape[1]] = part
    shape = thff.StateShape("half", rows // n, n, channels, order, 1, stride, stride, stride, stride, stride, stride)
    wide = {name: far[:, at:] for name, at in names.items()}
    got = {name: out[:, 64 * k:] for k, name in enumerate(("y", "dx", "ddelta", "dgate", "db", "dc"))}
    state, da = torch.empty_like(v["state"]), torch.empty_like(v["a"])
    saved = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
    workspace = torch.empty(shape.workspace_bytes(), dtype=torch.uint8, device="cuda")
    more = dict(d_skip=v["skip"], d_gate=wide["gate"], d_delta_bias=v["delta_bias"])
    calls = [(wide["x"], wide["delta"], v["a"], wide["b"], wide["c"], got["y"])]
    want = run("half", v)
    for d_saved in (None, saved):
        # A single step that saves nothing has a kernel of its own.
        thff.ThunderFFT_state_scan(shape, *calls[0], d_state_in=v["state"], d_state_out=state, d_saved=d_saved,
                                   d_workspace=workspace, **more)
        y = got["y"][:, :channels].reshape(want["y"].shape)
        if n > 1 or d_saved is not None:
            assert torch.equal(y, want["y"]) and torch.equal(state, want["state"])
        else:
            # The sum over the states in another order: two roundings of y's type and 16 of fp32's.
            bound = 2.0 ** -10 * want["y"].float().abs() + 2.0 ** -18 * want["y"].float().abs().max()
            assert ((y.float() - want["y"].float()).abs() <= bound).all()
    thff.ThunderFFT_state_scan_backward(
        shape, wide["dy"], wide["x"], wide["delta"], v["a"], wide["b"], wide["c"], saved, got["dx"], got["ddelta"], da, got["db"],
        got["dc"], d_dgate=got["dgate"], d_dstate_out=v["dstate"], d_workspace=workspace, **more)
    for name in ("dx", "ddelta", "dgate", "db", "dc"):
        part = want[name].reshape(rows, -1)
        assert torch.equal(got[name][:, :part.shape[1]], part), name
    assert torch.equal(da, want["da"])


def test_last_steps_of_far_sequences():
    """The tensor function on steps more than 2^24 elements apart, and their gradients, are as on dense ones."""
    v = values(32, "half", 3, 1, 40, 16)
    far = torch.empty(3, 1 << 25, dtype=torch.float16, device="cuda")
    names = ("x", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "state")
    at, leaves = 0, []
    for name in names:
        t = v[name]
        if t.dtype == torch.float16:
            row = t.flatten(1).shape[1]
            part = far[:, at:at + row].unflatten(1, t.shape[1:])
            part.copy_(t)
            t, at = part, at + row
        leaves.append(t.detach().requires_grad_())
    dense = [v[name].clone().requires_grad_() for name in names]
    dy = torch.empty(3, 1 << 25, dtype=torch.float16, device="cuda")[:, :40].unflatten(1, (1, 40))
    dy.copy_(v["dy"])
    for given, grad in ((leaves, dy), (dense, v["dy"])):
        torch.autograd.backward(thff.state_scan(*given), [grad, v["dstate"]])
    for name, one, other in zip(names, leaves, dense):
        assert torch.equal(one.grad, other.grad), name


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(1025, 1030, 3, 1), (513, 1030, 7, 2), (257, 1030, 16, 1), (263, 1030, 13, 2), (131, 1030, 24, 1),
                                  (65, 1030, 50, 1)], ids=str)
def test_one_token_of_many_sequences(T, size):
    """From 2^20 lanes on a lane has two sequences: an odd batch, strides, lengths of 0 and 1, and states in
    place in a larger pool, with slots that are none beside ones that are.  Some channels of each group against
    the formulas, as no channel depends on another."""
    batch, channels, order, groups = size
    v = values(33, T, batch, 1, channels, order, groups)
    gen = torch.Generator().manual_seed(34)
    states, all_of = batch + 37, torch.arange(batch)
    slots = torch.randperm(states, generator=gen)[:batch].to(torch.int32)
    slots[all_of % 5 == 3], slots[all_of % 11 == 7], slots[:2] = -1, states, -1
    some = (slots >= 0) & (slots < states)
    assert some[batch - 1] and (some[:-1:2] != some[1::2]).any()
    pool = torch.randn(states, channels, order, generator=gen).cuda()
    first = torch.where(some.view(-1, 1, 1).cuda(), pool[slots.clamp(0, states - 1).long().cuda()], 0.0)
    at = {k: placed(v[k], 3, 1)[0] for k in VALUES + SHARED}
    row = groups * order + 3
    shape = thff.StateShape(T, batch, 1, channels, order, groups, *(channels + 3,) * 3, row, row, channels + 3, states=states)
    few = torch.tensor([0, 1, 513, 514, 515, 516, 1028, 1029], device="cuda")
    for end in (None, (torch.arange(batch, device="cuda") % 3 != 1).to(torch.int32)):
        y, intact = placed(torch.full_like(v["x"], float("nan")), 3, 1)
        kept = torch.cat([pool, torch.full_like(pool[:1], GUARD)])
        print(f"{T} {size} lengths {end is not None}", flush=True)
        thff.ThunderFFT_state_scan(shape, at["x"], at["delta"], v["a"], at["b"], at["c"], y, d_skip=v["skip"], d_gate=at["gate"],
                                   d_delta_bias=v["delta_bias"], d_state_in=kept, d_state_out=kept, d_slots=slots.cuda(),
                                   d_lengths=end)
        assert intact() and torch.isfinite(y).all() and (kept[-1] == GUARD).all()
        free = torch.ones(states, dtype=torch.bool)
        free[slots[some].long()] = False
        assert torch.equal(kept[:-1][free.cuda()], pool[free.cuda()])
        mine = kept[slots[some].long().cuda()]
        if end is not None:
            assert torch.equal(mine[(end == 0)[some]], first[some.cuda()][(end == 0)[some]])
        for g in range(groups):
            c = few[few // (channels // groups) == g]
            want = oracle.state(T, v["x"][..., c], v["delta"][..., c], v["a"][c], v["b"][:, :, g:g + 1], v["c"][:, :, g:g + 1],
                                v["skip"][c], v["gate"][..., c], v["delta_bias"][c], first[:, c], end)
            oracle.check("y", y[..., c], want["y"])
            oracle.check("state", mine[:, c], tuple(t[some] for t in want["state"]))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("order", [4, 16, 40])
def test_segments_with_states_in_a_pool(T, order):
    """Prompts long enough for segments, in two calls, the states in place in rows of a pool: as each whole
    sequence, with a place that is none and lengths that end in any segment; other rows of the pool stay."""
    batch, n, channels = 5, 900, 24
    v = values(35, T, batch, n, channels, order)
    slots, rows = ends(6, 2, -1, 0, 5), [0, 1, 3, 4]
    pool = torch.full((8, channels, order), GUARD, device="cuda")
    pool[slots[rows].long()] = v["state"][rows]
    kept = pool.clone()
    lengths, at, y = torch.tensor([900, 700, 900, 30, 533]), 0, torch.empty_like(v["x"])
    for count in (500, 400):
        part = {k: v[k][:, at:at + count].contiguous() for k in VALUES + SHARED}
        shape = thff.StateShape(T, batch, count, channels, order, states=8)
        out = torch.empty_like(part["x"])
        assert shape.forward_bytes() > 0
        work = torch.full((shape.forward_bytes(),), 0xFF, dtype=torch.uint8, device="cuda")
        end = (lengths - at).clamp(0, count).to(torch.int32).cuda()
        thff.ThunderFFT_state_scan(shape, part["x"], part["delta"], v["a"], part["b"], part["c"], out, d_skip=v["skip"],
                                   d_gate=part["gate"], d_delta_bias=v["delta_bias"], d_state_in=pool, d_state_out=pool,
                                   d_slots=slots, d_lengths=end, d_workspace=work)
        y[:, at:at + count] = out
        at += count
    whole = oracle.state(T, v["x"], v["delta"], v["a"], v["b"], v["c"], v["skip"], v["gate"], v["delta_bias"], v["state"], lengths)
    for name, got in (("y", y), ("state", pool[slots.long()])):
        value, bound = whole[name]
        oracle.check(name, got[rows], (value[rows], bound[rows]))
    free = [r for r in range(8) if r not in (6, 2, 0, 5)]
    assert torch.equal(pool[free], kept[free])


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("low,high", [(-80.0, -20.0), (-20.0, -8.0), (-8.0, 0.0), (0.0, 20.0)])
def test_step_sizes(n, low, high):
    """dt alone: y is dt where the state is from zero, a = 0 and x = b = c = 1.  With u = 2^-24 and v = delta +
    delta_bias as fp32 has it: e = exp(-|v|) is off by 1.22 u |v| (the product and log2(e) as fp32 has it) and 2 u
    (exp2), relative to it and so to log(1 + e) at most; the logarithm of 1 + e rounded by 4 u, its product with
    log(2) and the sum with what the rounding lost by 1.1 u; what was lost, times 1 - e / 2 for 1 / (1 + e), by
    2.5 u: in all (1.25 |v| + 11) u of log(1 + e); and the sum with max(v, 0) by u of itself."""
    gen, u, channels = torch.Generator().manual_seed(36), 2.0 ** -24, 1 << 15
    delta = low + (high - low) * torch.rand(1, n, channels, generator=gen)
    bias = torch.randn(channels, generator=gen)
    shape = thff.StateShape("float", 1, n, channels, 1)
    for b in (None, bias):
        v = delta if b is None else (delta - b) + b
        given = (delta if b is None else delta - b).cuda()
        one, y = torch.ones_like(given), torch.empty_like(given)
        # Each step alone: b and c of the others are 0.
        for t in range(n):
            on = torch.zeros(1, n, 1, 1, device="cuda")
            on[:, t] = 1
            thff.ThunderFFT_state_scan(shape, one, given, torch.zeros(channels, 1, device="cuda"), on, on, y,
                                       d_delta_bias=None if b is None else b.cuda())
            got, w = y[:, t].cpu().double(), v[:, t].double()
            e = torch.log1p(torch.exp(-w.abs()))
            want = w.clamp(min=0) + e
            bound = (1.25 * w.abs() + 11) * u * e + u * want + 2.0 ** -126
            off = (got - want).abs() / bound
            print(f"n {n} step {t} {low} to {high}: {off.max().item():.3f} of the bound", flush=True)
            assert (off <= 1).all()


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(3, 1, 24, 5), (3, 18, 70, 16), (2, 45, 9, 40), (2, 700, 24, 4), (1, 1500, 12, 24)], ids=str)
def test_rates_of_the_lowest_value(T, size):
    """Rates that leave nothing of a state, at fp32's lowest value and at minus infinity: steps of 0 among the
    others and behind the ends keep the states, and gradients are finite."""
    v = values(37, T, *size)
    batch, n, channels, order = size
    v["a"][::2, ::2] = torch.finfo(torch.float32).min
    v["a"][1::3, 1] = torch.finfo(torch.float32).min
    # dt is exactly 0 where exp(delta + delta_bias) is; a small one is not.
    v["delta"][:, 3::7], v["delta"][:, 5::11] = -200, -300
    for lengths in (None, ends(*(n - 1 - n // 3 * b for b in range(batch)))):
        compare(T, v, lengths)
        got = run(T, v, lengths)
        below = dict(v, a=torch.where(v["a"] == torch.finfo(torch.float32).min, -float("inf"), v["a"]))
        other = run(T, below, lengths)
        for name in got:
            assert torch.equal(got[name], other[name]), name
    # The kernel of single steps.
    if n == 1:
        for a in (v["a"], below["a"]):
            for lengths in (None, ends(1, 0, 1)):
                delta = v["delta"].clone()
                delta[0, 0, ::2] = -200
                want = oracle.state(T, v["x"], delta, v["a"], v["b"], v["c"], v["skip"], v["gate"], v["delta_bias"], v["state"], lengths)
                y, state = thff.state_scan(v["x"], delta, a, v["b"], v["c"], v["skip"], v["gate"], v["delta_bias"], v["state"], lengths)
                oracle.check("y", y, want["y"])
                oracle.check("state", state, want["state"])


@pytest.mark.parametrize("n", [1, 45, 700])
def test_a_rate_that_is_none(n):
    """A NaN among the rates makes its channel's outputs, state and gradients NaN, and no other channel's."""
    v = values(38, "half", 2, n, 24, 16)
    clean = run("half", v)
    v["a"][5, 3] = float("nan")
    got = run("half", v)
    rest = torch.arange(24, device="cuda") != 5
    for name in ("y", "dx", "ddelta", "dgate"):
        assert torch.equal(got[name][..., rest], clean[name][..., rest]), name
    assert got["y"][..., 5].isnan().all() and got["dgate"][..., 5].isnan().all() and got["ddelta"][..., 5].isnan().all()
    assert torch.equal(got["state"][:, rest], clean["state"][:, rest]) and got["state"][:, 5, 3].isnan().all()
    assert torch.equal(got["da"][rest], clean["da"][rest]) and got["da"][5, 3].isnan()
    if n == 1:
        names = ("x", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "state")
        y, state = thff.state_scan(*(v[k] for k in names))
        assert y[..., 5].isnan().all() and state[:, 5, 3].isnan().all()
        assert torch.isfinite(y[..., rest]).all() and torch.isfinite(state[:, rest]).all()
