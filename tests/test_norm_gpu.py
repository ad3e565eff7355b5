"""Layer norm on the GPU against its definition in 64 bits: outputs and gradients, in all
types, from rows of one value to rows wider than registers hold, with strides, streams and
graphs."""
import pytest
import torch

import sequence_oracle as oracle
import thunderfft_amd as thff

pytestmark = pytest.mark.gpu
GUARD = -271.0
EPS = 1e-5


def values(seed, T, rows, cols):
    """x (rows of unlike offset and size), weight, bias, dy on the GPU."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    x = normal(rows, cols) * normal(rows, 1).exp() + normal(rows, 1)
    dt = oracle.TYPES[T]
    return (x.to(dt).cuda(), (1 + 0.2 * normal(cols)).cuda(), (0.2 * normal(cols)).cuda(), normal(rows, cols).to(dt).cuda())


def placed(v, stride, offset):
    """A copy of v with rows `stride` apart, `offset` elements into its buffer, and whether
    what is around the rows is as it was."""
    rows, cols = v.shape
    whole = torch.full((offset + rows * stride + 64,), GUARD, dtype=v.dtype, device="cuda")
    out = whole[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    out.copy_(v)

    def intact():
        around = whole.clone()
        around[offset:offset + rows * stride].view(rows, stride)[:, :cols] = GUARD
        return bool((around == GUARD).all())

    return out, intact


def run(T, x, weight, bias, dy, gap=0, offset=0, eps=EPS):
    rows, cols = x.shape
    stride = cols + gap
    print(f"{T} {rows} x {cols} gap {gap} offset {offset}", flush=True)
    nan = torch.full_like(x, float("nan"))
    (x, _), (dy, _), (y, y_ok), (dx, dx_ok) = (placed(v, stride, offset) for v in (x, dy, nan, nan))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    thff.ThunderFFT_layer_norm(T, x, weight, bias, eps, y, rows, cols, d_mean=mean, d_rstd=rstd, x_stride=stride,
                               y_stride=stride)
    assert y_ok()
    workspace = torch.full((thff.layer_norm_workspace_bytes(rows, cols),), 0xFF, dtype=torch.uint8, device="cuda")
    grads = torch.full((2 * cols + 8,), GUARD, device="cuda")
    dweight, dbias = grads[:cols], grads[cols + 4:2 * cols + 4]
    thff.ThunderFFT_layer_norm_backward(T, dy, x, mean, rstd, weight, dx, dweight, dbias, workspace, rows, cols,
                                        dy_stride=stride, x_stride=stride, dx_stride=stride)
    assert dx_ok() and (grads[cols:cols + 4] == GUARD).all() and (grads[2 * cols + 4:] == GUARD).all()
    return dict(y=y, dx=dx, dweight=dweight, dbias=dbias)


def compare(T, x, weight, bias, dy, eps=EPS, **how):
    got = run(T, x, weight, bias, dy, eps=eps, **how)
    want = oracle.norm(T, x, weight, bias, eps, dy)
    for name in want:
        oracle.check(name, got[name], want[name])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", [(1, 1), (5, 2), (3, 7), (1, 63), (9, 64), (2, 65), (1000, 16), (33, 255), (257, 256), (4, 257),
                                  (17, 511), (130, 512), (3, 777), (8, 1024), (6, 1025), (520, 2048), (5, 2049), (3, 4096),
                                  (2, 5001), (300, 8192), (3, 16384), (2, 20011), (1, 65536), (5000, 40)], ids=str)
def test_sizes(T, size):
    compare(T, *values(sum(size), T, *size))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("how", [dict(gap=1), dict(gap=8), dict(offset=1), dict(offset=4), dict(gap=24, offset=8)], ids=str)
def test_strides_and_offsets(T, how):
    for size in ((37, 200), (9, 1032), (5, 2047), (3, 9000)):
        compare(T, *values(3, T, *size), **how)


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_without_weights(T):
    x, weight, bias, dy = values(4, T, 40, 300)
    compare(T, x, None, None, dy)
    compare(T, x, weight, None, dy)
    compare(T, x, None, bias, dy)


@pytest.mark.parametrize("cols", [256, 777, 20011])
def test_gradients_wanted_singly(cols):
    """dweight or dbias alone, or neither, are as with both."""
    x, weight, bias, dy = values(5, "half", 300, cols)
    both = run("half", x, weight, bias, dy)
    rows = x.shape[0]
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    y, dx = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_layer_norm("half", x, weight, bias, EPS, y, rows, cols, d_mean=mean, d_rstd=rstd)
    workspace = torch.empty(thff.layer_norm_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    for w, b in ((True, False), (False, True), (False, False)):
        dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        dx.zero_()
        thff.ThunderFFT_layer_norm_backward("half", dy, x, mean, rstd, weight, dx, dw if w else None, db if b else None,
                                            workspace if w or b else None, rows, cols)
        assert torch.equal(dx, both["dx"])
        assert not w or torch.equal(dw, both["dweight"])
        assert not b or torch.equal(db, both["dbias"])


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_large_offsets_in_a_row(T):
    """A mean hundreds of deviations from zero costs its own rounding, and no cancellation."""
    x, weight, bias, dy = values(6, T, 20, 1000)
    compare(T, (x.float() * 0.1 + 64).to(x.dtype), weight, bias, dy)


@pytest.mark.parametrize("cols", [64, 777, 3000, 20011])
def test_constant_rows(cols):
    """No variance: y is the bias, and eps bounds the gradient; eps = 0 gives NaN there alone."""
    x, weight, bias, dy = values(7, "float", 6, cols)
    x[2] = 3.0
    compare("float", x, weight, bias, dy)
    y = torch.empty_like(x)
    thff.ThunderFFT_layer_norm("float", x, weight, bias, 0.0, y, 6, cols)
    bad = ~torch.isfinite(y)
    assert bad[2].all() and not bad[[0, 1, 3, 4, 5]].any()


@pytest.mark.parametrize("cols", [64, 777, 20011])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_non_finite_rows_stay_alone(cols, junk):
    x, weight, bias, dy = values(8, "half", 40, cols)
    y, z = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_layer_norm("half", x, weight, bias, EPS, y, 40, cols)
    x[7, cols // 2] = junk
    thff.ThunderFFT_layer_norm("half", x, weight, bias, EPS, z, 40, cols)
    rest = [r for r in range(40) if r != 7]
    assert torch.equal(y[rest], z[rest]) and z[7].isnan().any()


def test_no_rows():
    """No rows: the weights' gradients are zeros, whatever the workspace."""
    dw, db = torch.full((40,), GUARD, device="cuda"), torch.full((40,), GUARD, device="cuda")
    thff.ThunderFFT_layer_norm_backward("half", 0, 0, 0, 0, 0, 0, dw, db, 0, 0, 40)
    assert (dw == 0).all() and (db == 0).all()
    thff.ThunderFFT_layer_norm("half", 0, 0, 0, EPS, 0, 0, 40)


@pytest.mark.parametrize("size", [(4099, 520), (700, 20011)], ids=str)
def test_same_bits_each_time(size):
    args = values(9, "bfloat16", *size)
    first = run("bfloat16", *args)
    for _ in range(4):
        again = run("bfloat16", *args)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_rows_do_not_depend_on_each_other():
    """A row's bits are the same alone, in a batch, and at any place in it."""
    x, weight, bias, dy = values(10, "bfloat16", 1500, 520)
    whole = run("bfloat16", x, weight, bias, dy)
    for r in (0, 1, 700, 1499):
        one = run("bfloat16", x[r:r + 1], weight, bias, dy[r:r + 1])
        assert torch.equal(one["y"][0], whole["y"][r]) and torch.equal(one["dx"][0], whole["dx"][r])


def test_streams_and_graph_replays():
    """On a stream of its own, captured, and replayed with new inputs and eager calls between."""
    rows, cols = 3000, 520
    x, weight, bias, dy = values(11, "bfloat16", rows, cols)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    y, dx = torch.empty_like(x), torch.empty_like(x)
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    workspace = torch.empty(thff.layer_norm_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")

    def calls(stream):
        thff.ThunderFFT_layer_norm_async("bfloat16", x, weight, bias, EPS, y, rows, cols, d_mean=mean, d_rstd=rstd, stream=stream)
        thff.ThunderFFT_layer_norm_backward_async("bfloat16", dy, x, mean, rstd, weight, dx, dw, db, workspace, rows, cols,
                                                  stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls(side)
    torch.cuda.synchronize()
    want = run("bfloat16", x, weight, bias, dy)
    assert torch.equal(want["y"], y) and torch.equal(want["dweight"], dw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for k in range(4):
        new = values(50 + k, "bfloat16", rows, cols)
        for old, v in zip((x, weight, bias, dy), new):
            old.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = run("bfloat16", *new)
        for name, v in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
            assert torch.equal(want[name], v), (k, name)


def test_offsets_past_32_bits():
    rows, cols, stride = 5, 300, (1 << 30) + 8
    x, weight, bias, dy = values(12, "half", rows, cols)
    base = torch.empty((rows - 1) * stride + 4096, dtype=torch.float16, device="cuda")
    far = [base.as_strided((rows, cols), (stride, 1), 512 * k) for k in range(4)]
    far[0].copy_(x), far[1].copy_(dy)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    workspace = torch.empty(thff.layer_norm_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    thff.ThunderFFT_layer_norm("half", far[0], weight, bias, EPS, far[2], rows, cols, d_mean=mean, d_rstd=rstd,
                               x_stride=stride, y_stride=stride)
    thff.ThunderFFT_layer_norm_backward("half", far[1], far[0], mean, rstd, weight, far[3], dw, db, workspace, rows, cols,
                                        dy_stride=stride, x_stride=stride, dx_stride=stride)
    want = oracle.norm("half", x, weight, bias, EPS, dy)
    for name, v in (("y", far[2]), ("dx", far[3]), ("dweight", dw), ("dbias", db)):
        oracle.check(name, v, want[name])


def test_more_rows_than_one_launch_has_lanes():
    """2^30 rows of one value take several launches: each is its mean, so y is the bias."""
    rows = (1 << 30) + 5
    x = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    y = torch.full_like(x, float("nan"))
    mean, rstd = torch.full((rows,), GUARD, device="cuda"), torch.full((rows,), GUARD, device="cuda")
    bias = torch.full((1,), 0.75, device="cuda")
    thff.ThunderFFT_layer_norm("half", x, None, bias, 1.0, y, rows, 1, d_mean=mean, d_rstd=rstd)
    assert bool((y == 0.75).all()) and bool((mean == 1).all()) and bool((rstd == 1).all())


def test_gradients_against_differences():
    """As the recurrence's: a central difference of the float forward pass, off by its
    roundings and by the truncation that the same quotient in 64 bits has."""
    x, weight, bias, dy = values(13, "float", 12, 200)
    got = run("float", x, weight, bias, dy)
    want = oracle.norm("float", x, weight, bias, EPS, dy)
    eps = 2.0 ** -8

    def losses(ins):
        y = torch.empty_like(x)
        thff.ThunderFFT_layer_norm("float", ins[0], ins[1], ins[2], EPS, y, 12, 200)
        w = oracle.norm("float", *ins, EPS)["y"]
        d = dy.cpu().double()
        return float((y.cpu().double() * d).sum()), float((w[0] * d).sum()), float((w[1] * d.abs()).sum())

    gen = torch.Generator().manual_seed(1)
    for name, at in (("dx", 0), ("dweight", 1), ("dbias", 2)):
        ins = [x, weight, bias]
        v = torch.randn(ins[at].shape, generator=gen).cuda()
        up, down = list(ins), list(ins)
        up[at], down[at] = ins[at] + eps * v, ins[at] - eps * v
        step = (up[at].double() - down[at].double()).cpu()
        a, b = losses(up), losses(down)
        along = float((got[name].cpu().double() * step).sum())
        truncation = abs(a[1] - b[1] - float((want[name][0] * step).sum()))
        bound = a[2] + b[2] + truncation + float((want[name][1] * step.abs()).sum())
        assert abs(a[0] - b[0] - along) <= bound, (name, a[0] - b[0], along, bound)


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_tensor_function(T):
    """layer_norm with its gradients on three axes, on slices, and with a broadcast gradient."""
    x, weight, bias, dy = values(14, T, 60, 200)
    wide = torch.cat([x, x], -1).view(3, 20, 400)
    part = wide[..., 200:].detach().requires_grad_()
    w, b = weight.clone().requires_grad_(), bias.clone().requires_grad_()
    y = thff.layer_norm(part, w, b, EPS)
    y.backward(dy.view(3, 20, 200))
    want = oracle.norm(T, x, weight, bias, EPS, dy)
    for name, v in (("y", y), ("dx", part.grad)):
        oracle.check(name, v.reshape(60, 200), want[name])
    oracle.check("dweight", w.grad, want["dweight"])
    oracle.check("dbias", b.grad, want["dbias"])
    one = part[0, 0].detach().requires_grad_()
    thff.layer_norm(one, eps=EPS).backward(dy[:1, :1].expand(1, 200)[0])
    want = oracle.norm(T, x[:1], None, None, EPS, dy[:1, :1].expand(1, 200))
    oracle.check("dx", one.grad.unsqueeze(0), want["dx"])
    empty = torch.zeros(0, 40, device="cuda", dtype=oracle.TYPES[T], requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    thff.layer_norm(empty, w).sum().backward()
    assert (w.grad == 0).all() and empty.grad.shape == empty.shape


def test_tensor_function_refuses():
    x = torch.zeros(4, 8, device="cuda")
    for bad in (dict(weight=torch.ones(7, device="cuda")), dict(bias=torch.ones(8, device="cuda", dtype=torch.float16)),
                dict(weight=torch.ones(8)), dict(eps=-1.0), dict(x=x.double()), dict(x=torch.zeros(4, 0, device="cuda"))):
        with pytest.raises(ValueError):
            thff.layer_norm(**{"x": x, **bad})


@pytest.mark.parametrize("seed", range(24))
def test_drawn(seed):
    import random

    rng = random.Random(seed)
    T = rng.choice(list(oracle.TYPES))
    cols = int(2 ** rng.uniform(0, 14.5))
    if rng.random() < 0.5:
        cols = max(8, cols // 8 * 8)
    rows = max(1, min(int(2 ** rng.uniform(0, 13)), (1 << 21) // cols))
    compare(T, *values(seed, T, rows, cols), gap=rng.choice([0, 0, 3, 8]), offset=rng.choice([0, 0, 1, 8]))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("cols", [33, 60, 2500, 2560, 4104, 5120, 5121, 6001, 9000, 10240, 11001, 12288])
def test_rows_of_any_number_of_waves(T, cols):
    """Rows on both sides of what 1, 3, 5, 6, 10 and 12 waves hold, more of them than a pass takes."""
    for rows in (1, 1301):
        compare(T, *values(cols + rows, T, rows, cols), gap=cols % 3)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64], ids=str)
def test_tensor_function_whatever_the_default_type(default):
    """Statistics and weights' gradients are float32 where torch makes other tensors by default."""
    x, weight, bias, dy = values(15, "bfloat16", 60, 200)
    leaves = [v.detach().clone().requires_grad_() for v in (x, weight, bias)]
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        y = thff.layer_norm(*leaves)
        y.backward(dy)
    finally:
        torch.set_default_dtype(before)
    want = oracle.norm("bfloat16", x, weight, bias, EPS, dy)
    for name, v in (("y", y), ("dx", leaves[0].grad), ("dweight", leaves[1].grad), ("dbias", leaves[2].grad)):
        assert v.dtype == (torch.float32 if name in ("dweight", "dbias") else torch.bfloat16)
        oracle.check(name, v, want[name])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("cols", [16385, 40000])
def test_wide_rows_need_no_workspace(T, cols):
    """All gradients of rows past the widest that registers hold, without scratch memory."""
    rows = 270
    x, weight, bias, dy = values(17, T, rows, cols)
    mean, rstd = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
    dw, db = (torch.empty(cols, dtype=torch.float32, device="cuda") for _ in range(2))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_layer_norm(T, x, weight, bias, EPS, y, rows, cols, d_mean=mean, d_rstd=rstd)
    thff.ThunderFFT_layer_norm_backward(T, dy, x, mean, rstd, weight, dx, dw, db, None, rows, cols)
    want = oracle.norm(T, x, weight, bias, EPS, dy)
    for name, v in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
        oracle.check(name, v, want[name])


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_widest_held_rows(T):
    """On both sides of the widest row that registers hold, backward (16384) and forward (32768)."""
    for cols in (16383, 16384, 16385, 32767, 32768, 32769):
        compare(T, *values(cols, T, 2, cols))
