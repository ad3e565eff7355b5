"""The sequence operators next to the long convolutions, as cases that can be timed and checked.

The gated linear recurrence, per channel, with f = sigmoid(gate):

    h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  y[t] = h[t],  h[-1] = the state before the first step

and layer norm over the last axis.  T is the type of the values ("float", "half" or "bfloat16");
states, weights, biases and their gradients are float32.

op          what a pass does
step        one token of each of `batch` sequences, the states in a pool of `states` rows
scan        all `n` steps of each sequence, outputs and final states (a prompt)
scan_train  the same, then the gradients of x, the gate and the first state from those of
            the outputs and of the final states
norm        layer norm of `rows` rows of `cols` values
norm_train  the same, then the gradients of x, the weight and the bias

layout "last" is [batch][n][channels] and "first" is [batch][channels][n], as the convolutions
have it.  "fused" has x and the gate side by side in one projection's rows, and their gradients
alike.  "ragged" gives each sequence a length of its own up to n.
"""
import math

import torch

own = False

EPS = 1e-5
_DTYPE = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # One token for each of a few users: latency only.
        dict(name="step_bf16_8x1024", op="step", T="bfloat16", batch=8, channels=1024, states=16, fused=True),
        # One token for each of many users.
        dict(name="step_f16_256x4096", op="step", T="half", batch=256, channels=4096, states=300, fused=False),
        # Prompts of unlike lengths, an ordinary number of them.
        dict(name="scan_bf16_7x1000x2048_ragged", op="scan", T="bfloat16", layout="last", batch=7, n=1000, channels=2048,
             fused=True, ragged=True),
        # One very long document: few channels to share the work, a long way to go.
        dict(name="scan_bf16_1x65536x1024", op="scan", T="bfloat16", layout="last", batch=1, n=65536, channels=1024,
             fused=False, ragged=False),
        # The benchmark's long-convolution layer with a recurrence in the convolution's place.
        dict(name="scan_f16_256x64x4096_first", op="scan", T="half", layout="first", batch=256, n=4096, channels=64,
             fused=False, ragged=False),
        # A training step's share of one card, the largest.
        dict(name="scan_train_bf16_8x4096x2048", op="scan_train", T="bfloat16", layout="last", batch=8, n=4096, channels=2048,
             fused=True, ragged=False),
        # The convolution's layout in float at the ordinary size, odd batch, lengths of its own.
        dict(name="scan_train_f32_33x96x512_first", op="scan_train", T="float", layout="first", batch=33, n=512, channels=96,
             fused=False, ragged=True),
        # The rows of a few users' tokens: latency only.
        dict(name="norm_bf16_8x1024", op="norm", T="bfloat16", rows=8, cols=1024),
        # An ordinary prompt's rows, not a multiple of anything.
        dict(name="norm_f16_4099x2048", op="norm", T="half", rows=4099, cols=2048),
        # A training step's share of one card.
        dict(name="norm_train_bf16_32768x2048", op="norm_train", T="bfloat16", rows=32768, cols=2048),
        # A small model's step in float, odd both ways.
        dict(name="norm_train_f32_1001x777", op="norm_train", T="float", rows=1001, cols=777),
        # Wide rows.
        dict(name="norm_train_f16_2048x8192", op="norm_train", T="half", rows=2048, cols=8192),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A size of that range; two in three are multiples of 8 or 64, as models choose them."""
    v = _log_uniform(rng, low, high)
    m = rng.choice([1, 8, 64])
    return max(low, v // m * m)


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "norm", "norm_train", "norm_train"])
    T = rng.choice(["float", "half", "bfloat16"])
    if op == "step":
        batch = _log_uniform(rng, 1, 256)
        return dict(op=op, T=T, batch=batch, channels=_size(rng, 16, 4096), states=batch + rng.randint(0, 64), fused=rng.random() < 0.5)
    values = _log_uniform(rng, 1 << 12, 1 << (25 if T == "float" else 26))
    if op in ("norm", "norm_train"):
        cols = min(_size(rng, 16, 16384), values)
        return dict(op=op, T=T, rows=max(1, values // cols), cols=cols)
    channels = min(_size(rng, 16, 4096), values)
    n = min(_size(rng, 1, 65536), max(1, values // channels))
    layout = rng.choice(["last", "last", "first"])
    return dict(op=op, T=T, layout=layout, batch=min(1024, max(1, values // (channels * n))), n=n, channels=channels,
                fused=layout == "last" and rng.random() < 0.5, ragged=rng.random() < 0.3)


def _inputs(case, seed):
    """The inputs of a case, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPE[case["T"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(std).add_(mean)

    if case["op"] in ("norm", "norm_train"):
        rows, cols = case["rows"], case["cols"]
        # Rows of unlike offset and size, weights near one.
        x = normal(rows, cols).mul_(normal(rows, 1).exp_()).add_(normal(rows, 1))
        return dict(x=x.to(dtype), weight=normal(cols, mean=1.0, std=0.2), bias=normal(cols, std=0.2),
                    dy=normal(rows, cols).to(dtype) if case["op"] == "norm_train" else None)
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    shape = (batch, channels, n) if case.get("layout") == "first" else (batch, n, channels)
    # Gates that keep most of the state, as trained ones do, some for hundreds of steps.
    x, gate = normal(*shape).to(dtype), normal(*shape, mean=2.0, std=2.0).to(dtype)
    if case["fused"]:
        both = torch.cat([x, gate], -1)
        x, gate = both[..., :channels], both[..., channels:]
    got = dict(x=x, gate=gate, state=normal(case.get("states", batch), channels))
    if case["op"] == "step":
        # Each sequence in a row of the pool of its own; one place in eight of the batch is empty.
        slots = torch.randperm(case["states"], generator=gen, device="cuda")[:batch].to(torch.int32)
        empty = torch.arange(batch, device="cuda") % 8 == 7
        return dict(got, slots=torch.where(empty, -1, slots).to(torch.int32))
    got["lengths"] = (torch.randint(0, n + 1, (batch,), generator=gen, device="cuda").to(torch.int32)
                      if case["ragged"] else None)
    if case["op"] == "scan_train":
        got["dy"], got["dstate"] = normal(*shape).to(dtype), normal(batch, channels)
    return got


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        # The buffers that a user's program keeps for the results, and the plan.
        import thunderfft_amd as thff

        state["thff"] = thff
        x = state["x"]

        def empty(like):
            return torch.empty(like.shape, dtype=like.dtype, device="cuda")

        state["y"] = empty(x)
        if case["op"] in ("norm", "norm_train"):
            rows, cols = case["rows"], case["cols"]
            if case["op"] == "norm_train":
                state.update(mean=torch.empty(rows, device="cuda"), rstd=torch.empty(rows, device="cuda"),
                             dx=empty(x), dweight=torch.empty(cols, device="cuda"), dbias=torch.empty(cols, device="cuda"),
                             workspace=torch.empty(thff.layer_norm_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda"))
            return state
        channels = case["channels"]
        stride = 2 * channels if case["fused"] else None
        shape = thff.ScanShape(case["T"], case["batch"], case.get("n", 1), channels,
                               layout="channels_" + case.get("layout", "last"), x_stride=stride, gate_stride=stride,
                               states=case.get("states"))
        state["shape"] = shape
        state["state_out"] = state["state"].clone()
        state["workspace"] = torch.empty(shape.workspace_bytes(), dtype=torch.uint8, device="cuda")
        if case["op"] == "scan_train":
            state["saved"] = torch.empty(shape.saved_bytes(), dtype=torch.uint8, device="cuda")
            both = torch.empty(*x.shape[:-1], 2 * channels, dtype=x.dtype, device="cuda") if case["fused"] else None
            state["dx"] = both[..., :channels] if case["fused"] else empty(x)
            state["dgate"] = both[..., channels:] if case["fused"] else empty(x)
            state["dstate_in"] = torch.empty_like(state["state"])
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, thff, stream = s["case"], s["thff"], torch.cuda.current_stream()
    op = case["op"]
    if op == "norm":
        thff.ThunderFFT_layer_norm_async(case["T"], s["x"], s["weight"], s["bias"], EPS, s["y"], case["rows"], case["cols"],
                                         stream=stream)
        return s["y"]
    if op == "norm_train":
        thff.ThunderFFT_layer_norm_async(case["T"], s["x"], s["weight"], s["bias"], EPS, s["y"], case["rows"], case["cols"],
                                         d_mean=s["mean"], d_rstd=s["rstd"], stream=stream)
        thff.ThunderFFT_layer_norm_backward_async(case["T"], s["dy"], s["x"], s["mean"], s["rstd"], s["weight"], s["dx"],
                                                  s["dweight"], s["dbias"], s["workspace"], case["rows"], case["cols"],
                                                  stream=stream)
        return dict(y=s["y"], dx=s["dx"], dweight=s["dweight"], dbias=s["dbias"])
    thff.ThunderFFT_gated_scan_async(s["shape"], s["x"], s["gate"], s["y"], d_state_in=s["state"], d_state_out=s["state_out"],
                                     d_slots=s.get("slots"), d_lengths=s.get("lengths"), d_saved=s.get("saved"),
                                     d_workspace=s["workspace"], stream=stream)
    if op != "scan_train":
        return dict(y=s["y"], state=s["state_out"])
    thff.ThunderFFT_gated_scan_backward_async(s["shape"], s["dy"], s["x"], s["gate"], s["saved"], s["dx"], s["dgate"],
                                              d_dstate_out=s["dstate"], d_dstate_in=s["dstate_in"], d_lengths=s["lengths"],
                                              d_workspace=s["workspace"], stream=stream)
    return dict(y=s["y"], state=s["state_out"], dx=s["dx"], dgate=s["dgate"], dstate=s["dstate_in"])


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


def _run_plain(s):
    case = s["case"]
    op, dtype = case["op"], _DTYPE[case["T"]]
    x = s["x"].float()
    if op in ("norm", "norm_train"):
        centred = x - x.mean(-1, keepdim=True)
        rstd = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
        xh = centred * rstd
        y = (xh * s["weight"] + s["bias"]).to(dtype)
        if op == "norm":
            return y
        dy = s["dy"].float()
        g = dy * s["weight"]
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        return dict(y=y, dx=dx.to(dtype), dweight=(dy * xh).sum(0), dbias=dy.sum(0))
    gate = s["gate"].float()
    if op == "step":
        # An empty place starts from zero, and its state goes into a row that is dropped.
        active = (s["slots"] >= 0).unsqueeze(1)
        rows = torch.where(s["slots"] >= 0, s["slots"].long(), case["states"])
        pool = torch.cat([s["state"], torch.zeros_like(s["state"][:1])])
        h = torch.where(active, pool[rows], 0.0)
        h = torch.sigmoid(gate[:, 0]) * h + torch.sigmoid(-gate[:, 0]) * x[:, 0]
        return dict(y=h.unsqueeze(1).to(dtype), state=pool.index_copy(0, rows, h)[:-1])
    first = case["layout"] == "first"
    if first:
        x, gate = x.transpose(1, 2), gate.transpose(1, 2)
    f, rest = torch.sigmoid(gate), torch.sigmoid(-gate)
    u = rest * x
    valid = None
    if s["lengths"] is not None:
        # Past a sequence's end the state stays as it is.
        valid = (torch.arange(case["n"], device="cuda") < s["lengths"].unsqueeze(1)).unsqueeze(2)
        f, u = torch.where(valid, f, 1.0), torch.where(valid, u, 0.0)

    def laid_out(v):
        v = v if valid is None else torch.where(valid, v, 0.0)
        return (v.transpose(1, 2) if first else v).to(dtype).contiguous()

    h = _scan(f, u, s["state"])
    got = dict(y=laid_out(h), state=h[:, -1].contiguous())
    if op == "scan":
        return got
    dy = s["dy"].float()
    dy = dy.transpose(1, 2) if first else dy
    dy = dy if valid is None else torch.where(valid, dy, 0.0)
    after = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], 1)
    lam = _scan(after.flip(1), dy.flip(1), s["dstate"]).flip(1)
    before = torch.cat([s["state"].unsqueeze(1), h[:, :-1]], 1)
    got["dx"] = laid_out(rest * lam)
    got["dgate"] = laid_out(lam * (before - x) * f * rest)
    got["dstate"] = f[:, 0] * lam[:, 0]
    return got


def work(case):
    """Inputs read once, outputs written once.  Operations of an element: 8 for a step of the
    recurrence (4 of them its gate), 14 more for its gradients, 8 for the norm, 12 for its gradients."""
    op, size = case["op"], 4 if case["T"] == "float" else 2
    train = op in ("scan_train", "norm_train")
    if op in ("norm", "norm_train"):
        rows, cols = case["rows"], case["cols"]
        return dict(bytes=rows * cols * size * (4 if train else 2) + 4 * cols * (4 if train else 2),
                    flops=rows * cols * (20 if train else 8))
    batch, n, channels = case["batch"], case.get("n", 1), case["channels"]
    values = batch * n * channels
    return dict(bytes=values * size * (6 if train else 3) + 4 * batch * channels * (4 if train else 2),
                flops=values * (22 if train else 8))


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    x = s["x"].double()
    if op in ("norm", "norm_train"):
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        deviation = torch.sqrt(var + EPS)
        xh = (x - mean) / deviation
        weight = s["weight"].double()
        y = weight * xh + s["bias"].double()
        if op == "norm":
            return y
        dy = s["dy"].double()
        # y's derivative by x with the mean and the deviation as functions of x too.
        along = dy * weight
        dx = (along - (along.sum(-1, keepdim=True) + xh * (along * xh).sum(-1, keepdim=True)) / case["cols"]) / deviation
        return dict(y=y, dx=dx, dweight=torch.einsum("rc,rc->c", dy, xh), dbias=dy.sum(0))
    gate = s["gate"].double()
    if op == "step":
        slots = s["slots"].tolist()
        pool = s["state"].double()
        y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for b, row in enumerate(slots):
            f = 1 / (1 + torch.exp(-gate[b, 0]))
            h = x[b, 0] + f * ((pool[row] if row >= 0 else 0.0) - x[b, 0])
            y[b, 0] = h
            if row >= 0:
                pool[row] = h
        return dict(y=y, state=pool)
    first, batch, n, channels = case["layout"] == "first", case["batch"], case["n"], case["channels"]
    # Steps outermost, one after the other.
    order = (2, 0, 1) if first else (1, 0, 2)
    back = (1, 2, 0) if first else (1, 0, 2)
    x, gate = x.permute(order).contiguous(), gate.permute(order).contiguous()
    f = 1 / (1 + torch.exp(-gate))
    rest = 1 / (1 + torch.exp(gate))
    u = rest * x
    inside = torch.ones(n, batch, 1, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        inside = (torch.arange(n, device="cuda").unsqueeze(1) < s["lengths"]).unsqueeze(2)
        f.masked_fill_(~inside, 1.0)
        u.masked_fill_(~inside, 0.0)
    h = torch.empty(n + 1, batch, channels, dtype=torch.float64, device="cuda")
    h[0] = s["state"]
    for t in range(n):
        torch.addcmul(u[t], f[t], h[t], out=h[t + 1])

    def laid_out(v):
        return v.masked_fill(~inside, 0.0).permute(back).contiguous()

    got = dict(y=laid_out(h[1:]), state=h[n].clone())
    if op == "scan":
        return got
    dy = s["dy"].double().permute(order).masked_fill(~inside, 0.0)
    lam = torch.empty(n, batch, channels, dtype=torch.float64, device="cuda")
    carried = s["dstate"].double()
    for t in range(n - 1, -1, -1):
        torch.add(dy[t], carried, out=lam[t])
        carried = f[t] * lam[t]
    got["dx"] = laid_out(rest * lam)
    got["dgate"] = laid_out(lam * (h[:-1] - x) * f * rest)
    got["dstate"] = carried
    return got
