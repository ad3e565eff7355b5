"""The operators of a state space block, as cases that can be timed and checked.

A block takes the rows of a residual stream, norms them, projects them, mixes a few neighbouring
steps by a short causal convolution, and then all steps by a state space whose step sizes, inputs
and outputs depend on the data.  T is the type of the values ("float", "half" or "bfloat16").

conv    y[t] = silu(bias + sum_{k < width} weight[k] x[t - width + 1 + k]), per channel; the
        width - 1 values before the first step are a state, of type T.
state   dt = softplus(delta + delta_bias), for each channel and each of its `order` states
            h[t] = exp(dt a) h[t-1] + dt x[t] b[t],   y[t] = (sum over the states of c[t] h[t] + skip x[t]) silu(gate[t])
        with b and c shared by the channels of a group; the states are float32.
rms     s = x + residual, rounded to T, y = s / sqrt(mean(s^2) + eps) * weight over a row.

op            what a pass does
conv_step     one token of each of `batch` sequences, the states in a pool of `states` rows
conv          all `n` steps of each sequence, outputs and final states (a prompt)
conv_train    the same, then the gradients of x, the weights and the bias
state_step, state, state_train
              the same for the state space; gradients of all its inputs and weights
rms           the norm of `rows` rows of `cols` values, and the sums
rms_8bit      the same with an output of 8 bits (e4m3) with a float32 scale for every `block` columns
rms_train     the norm and the sums, then the gradients of x (the residual's is the same) and the weight

Values are [batch][n][channels].  "fused" has x (conv) or the gate (state) as one half of a
projection's rows, and b and c (state) side by side in a projection's rows, behind 32 values of
something else.  "ragged" gives each sequence a length of its own up to n.
"""
import math

import torch

own = False

EPS = 1e-5
LARGEST = 448.0  # of e4m3
_DTYPE = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # One token for each of a few users: latency only.
        dict(name="conv_step_bf16_8x2048", op="conv_step", T="bfloat16", batch=8, channels=2048, width=4, states=16, fused=True),
        # Prompts of unlike lengths, an ordinary number of them.
        dict(name="conv_f16_7x1000x2048_ragged", op="conv", T="half", batch=7, n=1000, channels=2048, width=4, fused=True,
             ragged=True),
        # A training step's share of one card.
        dict(name="conv_train_bf16_8x4096x2048", op="conv_train", T="bfloat16", batch=8, n=4096, channels=2048, width=4,
             fused=True, ragged=False),
        # One token for each of a few users: latency only.
        dict(name="state_step_bf16_8x1024", op="state_step", T="bfloat16", batch=8, channels=1024, order=16, groups=1, states=16,
             fused=True),
        # One token for each of many users.
        dict(name="state_step_f16_256x4096", op="state_step", T="half", batch=256, channels=4096, order=16, groups=1, states=300,
             fused=False),
        # Prompts of unlike lengths, an ordinary number of them.
        dict(name="state_bf16_7x1000x2048_ragged", op="state", T="bfloat16", batch=7, n=1000, channels=2048, order=16, groups=1,
             fused=True, ragged=True),
        # One very long document: few channels to share the work, a long way to go.
        dict(name="state_bf16_1x65536x1024", op="state", T="bfloat16", batch=1, n=65536, channels=1024, order=16, groups=1,
             fused=False, ragged=False),
        # A training step's share of one card, the largest.
        dict(name="state_train_bf16_8x4096x2048", op="state_train", T="bfloat16", batch=8, n=4096, channels=2048, order=16,
             groups=1, fused=True, ragged=False),
        # A small model's step in float: odd batch, an order that is no power of two, groups, lengths of their own.
        dict(name="state_train_f32_33x512x96_ragged", op="state_train", T="float", batch=33, n=512, channels=96, order=12,
             groups=2, fused=False, ragged=True),
        # The rows of a few users' tokens: latency only.
        dict(name="rms_bf16_8x1024", op="rms", T="bfloat16", rows=8, cols=1024),
        # An ordinary prompt's rows on their way to a product in 8 bits, not a multiple of anything.
        dict(name="rms_8bit_f16_4099x2048", op="rms_8bit", T="half", rows=4099, cols=2048, block=128),
        # A training step's share of one card.
        dict(name="rms_train_bf16_32768x2048", op="rms_train", T="bfloat16", rows=32768, cols=2048),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A size of that range; two in three are multiples of 8 or 64, as models choose them."""
    v = _log_uniform(rng, low, high)
    m = rng.choice([1, 8, 64])
    return max(low, v // m * m)


def draw(rng):
    op = rng.choice(["conv_step", "conv", "conv_train", "state_step", "state", "state", "state_train", "state_train", "rms",
                     "rms_8bit", "rms_train"])
    T = rng.choice(["float", "half", "bfloat16"])
    kind = op.split("_")[0]
    if kind == "rms":
        values = _log_uniform(rng, 1 << 12, 1 << (25 if T == "float" else 26))
        cols = min(_size(rng, 16, 16384), values)
        case = dict(op=op, T=T, rows=max(1, values // cols), cols=cols)
        if op == "rms_8bit":
            case["block"] = rng.choice([128, 128, cols])
        return case
    channels = _size(rng, 16, 4096)
    case = dict(op=op, T=T, channels=channels, fused=rng.random() < 0.5)
    if kind == "conv":
        case["width"] = rng.choice([2, 3, 4, 4])
    else:
        case["order"] = rng.choice([1, 4, 8, 12, 16, 16, 16, 16, 24, 32, 64])
        case["groups"] = rng.choice([g for g in (1, 1, 1, 2, 4, 8) if channels % g == 0])
    if op.endswith("step"):
        case["batch"] = _log_uniform(rng, 1, 256)
        case["states"] = case["batch"] + rng.randint(0, 64)
        return case
    values = _log_uniform(rng, 1 << 12, 1 << (25 if T == "float" else 26))
    if kind == "state":
        values = min(values, (1 << (29 if T == "float" else 30)) // case["order"])
    n = min(_size(rng, 1, 65536), max(1, values // channels))
    return dict(case, n=n, batch=min(1024, max(1, values // (channels * n))), ragged=rng.random() < 0.3)


def _inputs(case, seed):
    """The inputs of a case, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPE[case["T"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(std).add_(mean)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    kind, _, how = case["op"].partition("_")
    if kind == "rms":
        rows, cols = case["rows"], case["cols"]
        # A stream of residuals, larger than what a block adds to it, and weights near one.
        got = dict(x=normal(rows, cols).to(dtype), residual=normal(rows, cols).mul_(normal(rows, 1).exp_()).to(dtype),
                   weight=normal(cols, mean=1.0, std=0.2))
        if how == "train":
            got.update(dy=normal(rows, cols).to(dtype), dsum=normal(rows, cols).to(dtype))
        return got
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    got = dict(x=normal(batch, n, channels).to(dtype))
    if kind == "conv":
        width = case["width"]
        if case["fused"]:
            got["x"] = torch.cat([got["x"], normal(batch, n, channels).to(dtype)], -1)[..., :channels]
        got.update(weight=(uniform(channels, width) * 2 - 1) / width ** 0.5, bias=normal(channels, std=0.1),
                   state=normal(case.get("states", batch), width - 1, channels).to(dtype))
    else:
        order, groups = case["order"], case["groups"]
        gate = normal(batch, n, channels).to(dtype)
        if case["fused"]:
            gate = torch.cat([got["x"], gate], -1)[..., channels:]
        both = normal(batch, n, 32 + 2 * groups * order).to(dtype)
        b, c = both[..., 32:32 + groups * order], both[..., 32 + groups * order:]
        if not case["fused"]:
            b, c = b.contiguous(), c.contiguous()
        # Steps from a thousandth to a tenth, and states that forget at rates from one a unit up, as models are set up
        # with; trained ones differ from channel to channel.
        dt = torch.exp(uniform(channels) * math.log(100.0) + math.log(0.001))
        got.update(delta=normal(batch, n, channels, std=0.5).to(dtype), delta_bias=dt + torch.log(-torch.expm1(-dt)),
                   a=-(torch.arange(1, order + 1, device="cuda") * torch.exp(normal(channels, order, std=0.1))).contiguous(),
                   b=b, c=c, skip=normal(channels, mean=1.0, std=0.2), gate=gate,
                   state=normal(case.get("states", batch), channels, order))
    if how == "step":
        # Each sequence in a row of the pool of its own; one place in eight of the batch is empty.
        slots = torch.randperm(case["states"], generator=gen, device="cuda")[:batch].to(torch.int32)
        empty = torch.arange(batch, device="cuda") % 8 == 7
        return dict(got, slots=torch.where(empty, -1, slots).to(torch.int32))
    got["lengths"] = (torch.randint(0, n + 1, (batch,), generator=gen, device="cuda").to(torch.int32)
                      if case["ragged"] else None)
    if how == "train":
        got["dy"], got["dstate"] = normal(batch, n, channels).to(dtype), torch.randn(
            got["state"].shape, device="cuda", generator=gen).to(got["state"].dtype)
    return got


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        # The buffers that a user's program keeps for the results, and the plan.
        import thunderfft_amd as thff

        state["thff"] = thff
        _buffers(state, thff)
    return state


def _buffers(s, thff):
    case, x = s["case"], s["x"]
    kind, _, how = case["op"].partition("_")

    def like(v):
        return torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda")

    def dense(v):
        return torch.empty(v.shape, dtype=v.dtype, device="cuda")

    def scratch(count):
        return torch.empty(count, dtype=torch.uint8, device="cuda")

    if kind == "rms":
        rows, cols = case["rows"], case["cols"]
        s["sum"] = dense(x)
        if how == "8bit":
            s["q"] = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
            s["scales"] = torch.empty(rows, -(-cols // case["block"]), device="cuda")
            return
        s["y"] = dense(x)
        if how == "train":
            s.update(rstd=torch.empty(rows, device="cuda"), dx=dense(x), dweight=torch.empty(cols, device="cuda"),
                     workspace=scratch(thff.rms_norm_workspace_bytes(rows, cols)))
        return
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    s["y"], s["state_out"] = dense(x), s["state"].clone()
    if kind == "conv":
        shape = thff.ConvShape(case["T"], batch, n, channels, case["width"], silu=True, x_stride=x.stride(1),
                               states=case.get("states"))
    else:
        shape = thff.StateShape(case["T"], batch, n, channels, case["order"], groups=case["groups"],
                                gate_stride=s["gate"].stride(1), b_stride=s["b"].stride(1), c_stride=s["c"].stride(1),
                                states=case.get("states"))
    s["shape"] = shape
    s["workspace"] = scratch(shape.workspace_bytes())
    if how == "train":
        s.update(dstate_in=dense(s["state"]), dx=like(x))
        if kind == "conv":
            s.update(dweight=dense(s["weight"]), dbias=dense(s["bias"]))
        else:
            s["saved"] = scratch(shape.saved_bytes())
            s.update({"d" + name: like(s[name]) for name in ("delta", "a", "b", "c", "skip", "gate", "delta_bias")})


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, thff, stream = s["case"], s["thff"], torch.cuda.current_stream()
    op, T = case["op"], case["T"]
    if op == "rms_8bit":
        thff.ThunderFFT_rms_norm_8bit_async(T, s["x"], s["weight"], EPS, s["q"], s["scales"], case["rows"], case["cols"],
                                            case["block"], d_residual=s["residual"], d_sum=s["sum"], stream=stream)
        return dict(q=s["q"], scales=s["scales"], sum=s["sum"])
    if op in ("rms", "rms_train"):
        thff.ThunderFFT_rms_norm_async(T, s["x"], s["weight"], EPS, s["y"], case["rows"], case["cols"],
                                       d_residual=s["residual"], d_sum=s["sum"], d_rstd=s.get("rstd"), stream=stream)
        if op == "rms":
            return dict(y=s["y"], sum=s["sum"])
        thff.ThunderFFT_rms_norm_backward_async(T, s["dy"], s["sum"], s["rstd"], s["weight"], s["dx"], s["dweight"],
                                                s["workspace"], case["rows"], case["cols"], d_dsum=s["dsum"], stream=stream)
        return dict(y=s["y"], sum=s["sum"], dx=s["dx"], dweight=s["dweight"])
    how = dict(d_state_in=s["state"], d_state_out=s["state_out"], d_slots=s.get("slots"), d_lengths=s.get("lengths"),
               stream=stream)
    got = dict(y=s["y"], state=s["state_out"])
    if op in ("conv_step", "conv", "conv_train"):
        thff.ThunderFFT_short_conv_async(s["shape"], s["x"], s["weight"], s["bias"], s["y"], **how)
        if op == "conv_train":
            thff.ThunderFFT_short_conv_backward_async(
                s["shape"], s["dy"], s["x"], s["weight"], s["bias"], s["dx"], s["dweight"], s["dbias"], d_state_in=s["state"],
                d_dstate_out=s["dstate"], d_dstate_in=s["dstate_in"], d_lengths=s["lengths"], d_workspace=s["workspace"],
                stream=stream)
            got.update(dx=s["dx"], dweight=s["dweight"], dbias=s["dbias"], dstate=s["dstate_in"])
        return got
    thff.ThunderFFT_state_scan_async(s["shape"], s["x"], s["delta"], s["a"], s["b"], s["c"], s["y"], d_skip=s["skip"],
                                     d_gate=s["gate"], d_delta_bias=s["delta_bias"], d_saved=s.get("saved"),
                                     d_workspace=s["workspace"], **how)
    if op == "state_train":
        thff.ThunderFFT_state_scan_backward_async(
            s["shape"], s["dy"], s["x"], s["delta"], s["a"], s["b"], s["c"], s["saved"], s["dx"], s["ddelta"], s["da"], s["db"],
            s["dc"], d_skip=s["skip"], d_dskip=s["dskip"], d_gate=s["gate"], d_dgate=s["dgate"], d_delta_bias=s["delta_bias"],
            d_ddelta_bias=s["ddelta_bias"], d_dstate_out=s["dstate"], d_dstate_in=s["dstate_in"], d_lengths=s["lengths"],
            d_workspace=s["workspace"], stream=stream)
        got.update({name: s[name] for name in ("dx", "ddelta", "da", "db", "dc", "dskip", "dgate", "ddelta_bias")},
                   dstate=s["dstate_in"])
    return got


def _silu_slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def _pool_rows(s):
    """The pool with a row for empty places at its end, the rows of the sequences, and which are none."""
    active = s["slots"] >= 0
    pool = torch.cat([s["state"], torch.zeros_like(s["state"][:1])])
    return pool, torch.where(active, s["slots"].long(), s["case"]["states"]), active


def _valid(s):
    if s.get("lengths") is None:
        return None
    return (torch.arange(s["case"]["n"], device="cuda") < s["lengths"].unsqueeze(1)).unsqueeze(2)


def _run_plain(s):
    kind = s["case"]["op"].split("_")[0]
    return {"rms": _plain_rms, "conv": _plain_conv, "state": _plain_state}[kind](s)


def _plain_rms(s):
    case, dtype = s["case"], s["x"].dtype
    total = (s["x"].float() + s["residual"].float()).to(dtype)
    v = total.float()
    rstd = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = v * rstd
    y = xh * s["weight"]
    if case["op"] == "rms":
        return dict(y=y.to(dtype), sum=total)
    if case["op"] == "rms_8bit":
        rows, cols, block = case["rows"], case["cols"], case["block"]
        y = torch.nn.functional.pad(y, (0, -cols % block)).view(rows, -1, block)
        scales = (y.abs().amax(-1) / LARGEST).clamp(min=2.0 ** -126)
        q = (y / scales.unsqueeze(-1)).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn)
        return dict(q=q, scales=scales, sum=total)
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True)) + s["dsum"].float()
    return dict(y=y.to(dtype), sum=total, dx=dx.to(dtype), dweight=(dy * xh).sum(0))


def _plain_conv(s):
    case, dtype = s["case"], s["x"].dtype
    width, n = case["width"], case.get("n", 1)
    if case["op"] == "conv_step":
        # An empty place starts from zero, and its state goes into a row that is dropped.
        pool, rows, active = _pool_rows(s)
        before = torch.where(active.view(-1, 1, 1), pool[rows], 0.0)
    else:
        before = s["state"]
    whole = torch.cat([before, s["x"]], 1)
    v = whole.float()
    inner = s["bias"] + sum(v[:, k:k + n] * s["weight"][:, k] for k in range(width))
    valid = _valid(s)

    def laid_out(u):
        return (u if valid is None else torch.where(valid, u, 0.0)).to(dtype)

    y = laid_out(inner * torch.sigmoid(inner))
    if case["op"] == "conv_step":
        return dict(y=y, state=pool.index_copy(0, rows, whole[:, 1:])[:-1])
    ends = torch.full((case["batch"],), n, device="cuda") if valid is None else s["lengths"].long()
    # The last values of each sequence, which the next call starts from.
    last = ends.unsqueeze(1) + torch.arange(width - 1, device="cuda")
    last = last.unsqueeze(2).expand(-1, -1, case["channels"])
    got = dict(y=y, state=whole.gather(1, last))
    if case["op"] == "conv":
        return got
    dinner = s["dy"].float() * _silu_slope(inner)
    dinner = dinner if valid is None else torch.where(valid, dinner, 0.0)
    dwhole = torch.zeros_like(v).scatter_(1, last, s["dstate"].float())
    for k in range(width):
        dwhole[:, k:k + n] += dinner * s["weight"][:, k]
    got["dx"], got["dstate"] = laid_out(dwhole[:, width - 1:]), dwhole[:, :width - 1].to(dtype)
    if valid is not None:
        # Values behind an end are used nowhere, whatever they hold.
        used = torch.arange(v.shape[1], device="cuda") < ends.unsqueeze(1) + width - 1
        v = torch.where(used.unsqueeze(2), v, 0.0)
    got["dweight"] = torch.stack([(dinner * v[:, k:k + n]).sum((0, 1)) for k in range(width)], 1)
    got["dbias"] = dinner.sum((0, 1))
    return got


def _scan(a, b, first):
    """h[t] = a[t] h[t-1] + b[t] over axis 1, h[-1] = first, by doubling: after each round h[t]
    holds the terms of twice as many steps, and a[t] the product of as many factors."""
    b = torch.cat([torch.addcmul(b[:, :1], a[:, :1], first.unsqueeze(1)), b[:, 1:]], 1)
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], torch.addcmul(b[:, step:], a[:, step:], b[:, :-step])], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_state(s):
    case, dtype = s["case"], s["x"].dtype
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    order, groups = case["order"], case["groups"]
    valid = _valid(s)

    def inside(u):
        return u if valid is None else torch.where(valid, u, 0.0)

    def grouped(u):
        """(batch, n, channels, order) of b or c, which the channels of a group share."""
        return u.float().view(batch, n, groups, 1, order).expand(-1, -1, -1, channels // groups, -1).reshape(
            batch, n, channels, order)

    x, gate = inside(s["x"].float()), s["gate"].float()
    raw = s["delta"].float() + s["delta_bias"]
    # Past a sequence's end the state stays as it is.
    dt = inside(torch.clamp(raw, min=0.0) + torch.log1p(torch.exp(-raw.abs())))
    a = torch.exp(dt.unsqueeze(-1) * s["a"])
    b, c = grouped(inside(s["b"].float())), grouped(inside(s["c"].float()))
    u = (dt * x).unsqueeze(-1) * b
    if case["op"] == "state_step":
        # An empty place starts from zero, and its state goes into a row that is dropped.
        pool, rows, active = _pool_rows(s)
        h = (a[:, 0] * torch.where(active.view(-1, 1, 1), pool[rows], 0.0) + u[:, 0]).unsqueeze(1)
        state = pool.index_copy(0, rows, h[:, 0])[:-1]
    else:
        h = _scan(a, u, s["state"])
        state = h[:, -1].contiguous()
    inner = (h * c).sum(-1) + s["skip"] * x
    z = gate * torch.sigmoid(gate)
    got = dict(y=inside(inner * z).to(dtype), state=state)
    if case["op"] != "state_train":
        return got
    del u
    dy = inside(s["dy"].float())
    got["dgate"] = inside(dy * inner * _silu_slope(gate)).to(dtype)
    dinner = inside(dy * z)
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    lam = _scan(after.flip(1), (dinner.unsqueeze(-1) * c).flip(1), s["dstate"]).flip(1)
    del after
    got["dc"] = (dinner.unsqueeze(-1) * h).view(batch, n, groups, -1, order).sum(3).view(batch, n, -1).to(dtype)
    h = torch.cat([s["state"].unsqueeze(1), h[:, :-1]], 1)
    # Of the exponents dt a, and of the inputs dt x b.
    decayed = lam * a
    got["dstate"] = decayed[:, 0].contiguous()
    decayed *= h
    del h
    du = (lam * b).sum(-1)
    lam *= (dt * x).unsqueeze(-1)
    got["db"] = lam.view(batch, n, groups, -1, order).sum(3).view(batch, n, -1).to(dtype)
    got["dx"] = inside(du * dt + dinner * s["skip"]).to(dtype)
    draw_ = inside((du * x + (decayed * s["a"]).sum(-1)) * torch.sigmoid(raw))
    got["ddelta"], got["ddelta_bias"] = draw_.to(dtype), draw_.sum((0, 1))
    got["da"] = (decayed * dt.unsqueeze(-1)).sum((0, 1))
    got["dskip"] = (dinner * x).sum((0, 1))
    return got


def work(case):
    """Inputs read once, outputs written once.  Operations: of the norm 6 a value, 10 more for its gradients; of the
    convolution 2 a tap and 5, and 4 a tap and 10 more; of the state space, for each state of each value, 6 (the
    exponent, the input, two for the state, two for the output) and 17 more for its gradients, and 12 and 25 more a
    value."""
    op, size = case["op"], 4 if case["T"] == "float" else 2
    kind, _, how = op.partition("_")
    train = how == "train"
    if kind == "rms":
        rows, cols = case["rows"], case["cols"]
        values = rows * cols
        if how == "8bit":
            return dict(bytes=values * (3 * size + 1) + 4 * cols + 4 * rows * -(-cols // case["block"]), flops=8 * values)
        return dict(bytes=values * size * (7 if train else 4) + 4 * cols * (2 if train else 1), flops=values * (16 if train else 6))
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    values = batch * n * channels
    if kind == "conv":
        width = case["width"]
        weights, states = 4 * channels * (width + 1), batch * channels * (width - 1) * size
        return dict(bytes=values * size * (4 if train else 2) + weights * (2 if train else 1) + states * (4 if train else 2),
                    flops=values * (2 * width + 5 + (4 * width + 10 if train else 0)))
    order = case["order"]
    shared = 2 * batch * n * case["groups"] * order
    weights, states = 4 * channels * (order + 2), 4 * batch * channels * order
    return dict(bytes=(values * (8 if train else 4) + shared * (2 if train else 1)) * size + weights * (2 if train else 1) +
                states * (4 if train else 2),
                flops=values * (order * (23 if train else 6) + (37 if train else 12)))


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["op"].split("_")[0]
    return {"rms": _exact_rms, "conv": _exact_conv, "state": _exact_state}[kind](case, s)


def _exact_rms(case, s):
    dtype, cols = s["x"].dtype, case["cols"]
    total = (s["x"].double() + s["residual"].double()).to(dtype)
    v, weight = total.double(), s["weight"].double()
    size = torch.sqrt(torch.einsum("rc,rc->r", v, v) / cols + EPS).unsqueeze(1)
    y = weight * v / size
    if case["op"] == "rms":
        return dict(y=y, sum=total.double())
    if case["op"] == "rms_8bit":
        scales, q = [], []
        for part in y.split(case["block"], 1):
            scales.append(part.abs().max(1, keepdim=True).values / LARGEST)
            q.append((part / scales[-1]).float().to(torch.float8_e4m3fn))
        return dict(q=torch.cat([p.float() for p in q], 1), scales=torch.cat(scales, 1), sum=total.double())
    along = s["dy"].double() * weight
    # y's derivative by v with the root as a function of v too.
    dx = along / size - v * (along * v).sum(1, keepdim=True) / (cols * size ** 3) + s["dsum"].double()
    return dict(y=y, sum=total.double(), dx=dx, dweight=(s["dy"].double() * v / size).sum(0))


def _ends(case, s):
    return s["lengths"].tolist() if s.get("lengths") is not None else [case.get("n", 1)] * case["batch"]


def _exact_conv(case, s):
    """Sequence by sequence, each over its own steps alone."""
    width, n, channels = case["width"], case.get("n", 1), case["channels"]
    step, train = case["op"] == "conv_step", case["op"] == "conv_train"
    weight, bias = s["weight"].double(), s["bias"].double()
    slots = s["slots"].tolist() if step else range(case["batch"])
    state = s["state"].double()
    y = torch.zeros(case["batch"], n, channels, dtype=torch.float64, device="cuda")
    got = dict(y=y, state=state.clone())
    if train:
        got.update(dx=torch.zeros_like(y), dstate=torch.zeros_like(state), dweight=torch.zeros_like(weight),
                   dbias=torch.zeros_like(bias))
    for i, (row, end) in enumerate(zip(slots, _ends(case, s))):
        if end == 0:
            if train:
                got["dstate"][i] = s["dstate"][i].double()
            continue
        before = state[row] if row >= 0 else torch.zeros_like(state[0])
        v = torch.cat([before, s["x"][i, :end].double()])
        windows = v.unfold(0, width, 1)  # (end, channels, width)
        inner = torch.einsum("tck,ck->tc", windows, weight) + bias
        opened = 1 / (1 + torch.exp(-inner))
        y[i, :end] = inner * opened
        if row >= 0:
            got["state"][row] = v[end:]
        if train:
            d = s["dy"][i, :end].double() * (opened + inner * opened * (1 - opened))
            got["dweight"] += torch.einsum("tc,tck->ck", d, windows)
            got["dbias"] += d.sum(0)
            dv = torch.zeros_like(v)
            dv[end:] = s["dstate"][i].double()
            for k in range(width):
                dv[k:k + end] += d * weight[:, k]
            got["dstate"][i], got["dx"][i, :end] = dv[:width - 1], dv[width - 1:]
    return got


def _exact_state(case, s):
    """Step by step from the definition, steps outermost."""
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    order, groups = case["order"], case["groups"]
    each = channels // groups
    train = case["op"] == "state_train"
    if n * (15 if train else 5) > 1_200_000:
        return None

    def steps(v, *last):
        return v.double().transpose(0, 1).reshape(n, batch, *last)

    x, delta, gate = (steps(s[name], channels) for name in ("x", "delta", "gate"))
    b, c = (steps(s[name], groups, 1, order) for name in ("b", "c"))
    inside = torch.ones(n, batch, 1, dtype=torch.bool, device="cuda")
    if s.get("lengths") is not None:
        inside = (torch.arange(n, device="cuda").unsqueeze(1) < s["lengths"]).unsqueeze(2)
    raw = delta + s["delta_bias"].double()
    dt = torch.logaddexp(raw, torch.zeros_like(raw)).masked_fill(~inside, 0.0)
    u = dt * x
    a, skip = s["a"].double(), s["skip"].double()
    if case["op"] == "state_step":
        first = torch.zeros(batch, channels, order, dtype=torch.float64, device="cuda")
        for i, row in enumerate(s["slots"].tolist()):
            if row >= 0:
                first[i] = s["state"][row]
    else:
        first = s["state"].double()
    # All states are kept only where the gradients need them.
    hs = torch.empty(n if train else 0, batch, channels, order, dtype=torch.float64, device="cuda")
    inner = torch.empty(n, batch, channels, dtype=torch.float64, device="cuda")
    h = first
    for t in range(n):
        if train:
            hs[t] = h
        h = torch.exp(dt[t].unsqueeze(-1) * a) * h
        h.view(batch, groups, each, order).addcmul_(u[t].view(batch, groups, each, 1), b[t])
        torch.sum(h.view(batch, groups, each, order) * c[t], -1, out=inner[t].view(batch, groups, each))
    inner += skip * x
    opened = 1 / (1 + torch.exp(-gate))

    def back(v):
        return v.masked_fill(~inside, 0.0).transpose(0, 1).contiguous()

    got = dict(y=back(inner * gate * opened), state=h)
    if case["op"] == "state_step":
        got["state"] = s["state"].double()
        for i, row in enumerate(s["slots"].tolist()):
            if row >= 0:
                got["state"][row] = h[i]
    if not train:
        return got
    dy = steps(s["dy"], channels).masked_fill(~inside, 0.0)
    got["dgate"] = back(dy * inner * (opened + gate * opened * (1 - opened)))
    del inner
    dinner = dy * gate * opened
    du, dexponent = torch.empty_like(x), torch.empty_like(x)
    db, dc = (torch.empty(n, batch, groups, order, dtype=torch.float64, device="cuda") for _ in range(2))
    da, lam = torch.zeros_like(a), s["dstate"].double()
    for t in range(n - 1, -1, -1):
        keep = torch.exp(dt[t].unsqueeze(-1) * a)
        now = keep * hs[t]
        new = now.view(batch, groups, each, order) + u[t].view(batch, groups, each, 1) * b[t]
        along = dinner[t].view(batch, groups, each, 1)
        dc[t] = (along * new).sum(2)
        lam = (lam.view(batch, groups, each, order) + along * c[t]).view(batch, channels, order)
        du[t] = (lam.view(batch, groups, each, order) * b[t]).sum(-1).view(batch, channels)
        db[t] = (lam * u[t].unsqueeze(-1)).view(batch, groups, each, order).sum(2)
        now *= lam
        dexponent[t] = (now * a).sum(-1)
        da.add_(torch.einsum("bco,bc->co", now, dt[t]))
        lam = lam * keep
    draw_ = ((du * x + dexponent) / (1 + torch.exp(-raw))).masked_fill(~inside, 0.0)
    got.update(dx=back(du * dt + dinner * skip), ddelta=back(draw_), ddelta_bias=draw_.sum((0, 1)), da=da,
               db=back(db.view(n, batch, -1)), dc=back(dc.view(n, batch, -1)),
               dskip=(dinner * x).masked_fill(~inside, 0.0).sum((0, 1)), dstate=lam)
    return got
