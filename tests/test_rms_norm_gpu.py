"""Root-mean-square norm on the GPU against its definition in 64 bits: outputs, sums with a residual,
gradients and 8-bit outputs, in all types, from rows of one value to rows wider than registers hold."""
import pytest
import torch

import block_oracle as oracle
import thunderfft_amd as thff

pytestmark = pytest.mark.gpu
GUARD = -271.0
EPS = 1e-5
SIZES = [(1, 1), (5, 2), (3, 7), (1, 63), (9, 64), (2, 65), (1000, 16), (33, 255), (257, 256), (4, 257), (17, 511), (130, 512),
         (3, 777), (8, 1024), (6, 1025), (520, 2048), (5, 2049), (3, 4096), (2, 5001), (30, 8192), (3, 16384), (2, 20011),
         (1, 65536), (5000, 40)]


def values(seed, T, rows, cols):
    """x, residual, weight, dy, dsum on the GPU."""
    gen, dt = torch.Generator().manual_seed(seed), oracle.TYPES[T]

    def normal(*s):
        return torch.randn(*s, generator=gen)

    return (normal(rows, cols).to(dt).cuda(), (normal(rows, cols) * normal(rows, 1).exp()).to(dt).cuda(), (1 + 0.2 * normal(cols)).cuda(),
            normal(rows, cols).to(dt).cuda(), normal(rows, cols).to(dt).cuda())


def placed(v, stride, offset):
    """A copy of v with rows `stride` apart, `offset` elements into its buffer, and whether what is
    around the rows is as it was."""
    rows, cols = v.shape
    whole = torch.full((offset + rows * stride + 64,), GUARD, dtype=v.dtype, device="cuda")
    out = whole[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    out.copy_(v)

    def intact():
        around = whole.clone()
        around[offset:offset + rows * stride].view(rows, stride)[:, :cols] = GUARD
        return bool((around == GUARD).all())

    return out, intact


def run(T, x, residual, weight, dy, dsum, gap=0, offset=0):
    rows, cols = x.shape
    stride = cols + gap
    print(f"{T} {rows} x {cols} gap {gap} offset {offset}", flush=True)
    nan = torch.full_like(x, float("nan"))
    (x, _), (dy, _), (y, y_ok), (dx, dx_ok), (total, sum_ok) = (placed(v, stride, offset) for v in (x, dy, nan, nan, nan))
    residual, dsum = (None if v is None else placed(v, stride, offset)[0] for v in (residual, dsum))
    rstd = torch.empty(rows, device="cuda")
    thff.ThunderFFT_rms_norm(T, x, weight, EPS, y, rows, cols, d_residual=residual, d_sum=total, d_rstd=rstd, x_stride=stride,
                             residual_stride=stride, y_stride=stride, sum_stride=stride)
    assert y_ok() and sum_ok()
    workspace = torch.full((thff.rms_norm_workspace_bytes(rows, cols),), 0xFF, dtype=torch.uint8, device="cuda")
    grads = torch.full((cols + 4,), GUARD, device="cuda")
    thff.ThunderFFT_rms_norm_backward(T, dy, total, rstd, weight, dx, grads, workspace, rows, cols, d_dsum=dsum, dy_stride=stride,
                                      sum_stride=stride, dsum_stride=stride, dx_stride=stride)
    assert dx_ok() and (grads[cols:] == GUARD).all()
    return dict(y=y, sum=total, dx=dx, dweight=grads[:cols], rstd=rstd)


def compare(T, x, residual, weight, dy, dsum, **how):
    got = run(T, x, residual, weight, dy, dsum, **how)
    want = oracle.rms(T, x, weight, EPS, residual, dy, dsum)
    for name in want:
        oracle.check(name, got[name], want[name])


def run8(T, x, residual, weight, block, gap=0, offset=0):
    rows, cols = x.shape
    stride = cols + gap
    print(f"8 bit {T} {rows} x {cols} block {block} gap {gap} offset {offset}", flush=True)
    (x, _), (total, sum_ok) = (placed(v, stride, offset) for v in (x, torch.full_like(x, float("nan"))))
    residual = None if residual is None else placed(residual, stride, offset)[0]
    q = torch.full((offset + rows * stride + 64,), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows * -(-cols // block) + 4,), GUARD, device="cuda")
    at = q[offset:]
    thff.ThunderFFT_rms_norm_8bit(T, x, weight, EPS, at, scales, rows, cols, block, d_residual=residual, d_sum=total, x_stride=stride,
                                  residual_stride=stride, q_stride=stride, sum_stride=stride)
    got = at[:rows * stride].view(rows, stride)[:, :cols].clone()
    at[:rows * stride].view(rows, stride)[:, :cols] = 0x55
    assert (q == 0x55).all() and (scales[rows * -(-cols // block):] == GUARD).all() and sum_ok()
    return got.view(torch.float8_e4m3fn), scales[:rows * -(-cols // block)].view(rows, -1), total


def compare8(T, x, residual, weight, block, **how):
    q, scales, total = run8(T, x, residual, weight, block, **how)
    rows, cols = x.shape
    want, (y, off) = oracle.rms_8bit(T, x.cpu(), weight, EPS, block, None if residual is None else residual.cpu())
    oracle.check("scales", scales, want)
    s = scales.cpu().double().repeat_interleave(block, 1)[:, :cols]
    value = q.cpu().float().double() * s
    # Half a step of q: 2^-4 of itself, 2^-10 of a scale for the least; the quotient is off by 3 u.
    bound = off + (y.abs() + off) * 2.0 ** -4 + s * 2.0 ** -10 + 3 * oracle.U * y.abs()
    assert ((value - y).abs() <= bound).all()
    # The largest of a block is 448 but for the roundings of the scale and the quotient.
    wide = torch.nn.functional.pad(q.cpu().float().abs(), (0, -cols % block)).view(rows, -1, block)
    assert (wide.amax(2) == 448).all()
    if residual is not None:
        assert torch.equal(total, (x.double() + residual.double()).to(x.dtype))


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(T, size):
    x, residual, weight, dy, dsum = values(sum(size), T, *size)
    compare(T, x, residual, weight, dy, dsum)
    compare(T, x, None, weight, dy, None)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_8bit_sizes(T, size):
    x, residual, weight, *_ = values(sum(size), T, *size)
    compare8(T, x, residual, weight, 128)
    compare8(T, x, None, weight, size[1])


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("how", [dict(gap=1), dict(gap=8), dict(offset=1), dict(offset=4), dict(gap=24, offset=8)], ids=str)
def test_strides_and_offsets(T, how):
    for size in ((37, 200), (9, 1032), (5, 2047), (3, 9000), (2, 40001)):
        args = values(3, T, *size)
        compare(T, *args, **how)
        compare8(T, *args[:3], 128, **how)


@pytest.mark.parametrize("T", list(oracle.TYPES))
def test_without_weights(T):
    x, residual, weight, dy, dsum = values(4, T, 40, 300)
    compare(T, x, residual, None, dy, dsum)
    compare(T, x, residual, weight, dy, None)
    compare(T, x, None, weight, dy, dsum)
    compare8(T, x, None, None, 128)


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("cols", [7, 77, 200, 2047, 9001, 20011, 40001])
def test_sums_in_the_residuals_place(T, cols):
    """The residuals may be replaced by the sums: the same bits as with a buffer of their own."""
    x, residual, weight, dy, dsum = values(5, T, 65, cols)
    apart = run(T, x, residual, weight, dy, dsum)
    y, kept = torch.empty_like(x), residual.clone()
    thff.ThunderFFT_rms_norm(T, x, weight, EPS, y, 65, cols, d_residual=kept, d_sum=kept)
    assert torch.equal(y, apart["y"]) and torch.equal(kept, apart["sum"])
    for block in (128, cols):
        q, scales, _ = run8(T, x, residual, weight, block)
        other, kept = torch.empty(65, cols, dtype=torch.uint8, device="cuda"), residual.clone()
        more = torch.empty_like(scales)
        thff.ThunderFFT_rms_norm_8bit(T, x, weight, EPS, other, more, 65, cols, block, d_residual=kept, d_sum=kept)
        assert torch.equal(other, q.view(torch.uint8)) and torch.equal(more, scales) and torch.equal(kept, apart["sum"])


@pytest.mark.parametrize("cols", [256, 777, 20011])
def test_outputs_wanted_singly(cols):
    """Without the sums, the statistics or the weight's gradient the rest is as with them."""
    x, residual, weight, dy, dsum = values(6, "half", 300, cols)
    whole = run("half", x, residual, weight, dy, dsum)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_rms_norm("half", x, weight, EPS, y, 300, cols, d_residual=residual)
    assert torch.equal(y, whole["y"])
    thff.ThunderFFT_rms_norm_backward("half", dy, whole["sum"], whole["rstd"], weight, dx, None, None, 300, cols, d_dsum=dsum)
    assert torch.equal(dx, whole["dx"])


@pytest.mark.parametrize("size", [(700, 64), (90, 777), (64, 2048), (7, 20011), (5, 40001)], ids=str)
def test_8bit_is_the_rounded_quotient(size):
    """Each bit of it: the scale is the block's largest over 448, q the value over the scale, rounded once."""
    x, residual, weight, *_ = values(14, "float", *size)
    rows, cols = size
    y = run("float", x, residual, weight, x, None)["y"].cpu()
    for block in (128, cols):
        q, scales, _ = run8("float", x, residual, weight, block)
        padded = torch.nn.functional.pad(y, (0, -cols % block)).view(rows, -1, block)
        assert torch.equal(scales.cpu(), padded.abs().amax(2) / 448)
        want = (y / scales.cpu().repeat_interleave(block, 1)[:, :cols]).to(torch.float8_e4m3fn)
        assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("cols", [64, 130, 777, 20011, 40001])
def test_zero_rows(cols):
    """Rows of zeros: y is 0, q is 0 with the least scale; with eps = 0 they are NaN, and no others."""
    x, residual, weight, dy, dsum = values(7, "float", 6, cols)
    x[2] = 0
    residual[2] = 0
    compare("float", x, residual, weight, dy, dsum)
    for block in (128, cols):
        q, scales, _ = run8("float", x, residual, weight, block)
        assert (q[2].float() == 0).all() and (scales[2] == 2.0 ** -126).all()
    y = torch.empty_like(x)
    thff.ThunderFFT_rms_norm("float", x, weight, 0.0, y, 6, cols)
    bad = ~torch.isfinite(y)
    assert bad[2].all() and not bad[[0, 1, 3, 4, 5]].any()


@pytest.mark.parametrize("cols", [300, 2048, 20011])
def test_a_block_of_zeros(cols):
    """A block of 128 zeros among others has the least scale and zeros; the others are as without it."""
    x, _, weight, *_ = values(8, "half", 5, cols)
    x[3, 128:256] = 0
    q, scales, _ = run8("half", x, None, weight, 128)
    assert (q[3, 128:256].float() == 0).all() and scales[3, 1] == 2.0 ** -126
    assert (scales[[0, 1, 2, 4]] > 2.0 ** -126).all() and scales[3, 0] > 2.0 ** -126 and scales[3, 2] > 2.0 ** -126


@pytest.mark.parametrize("cols", [64, 777, 20011, 40001])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_non_finite_rows_stay_alone(cols, junk):
    x, residual, weight, *_ = values(9, "half", 40, cols)
    y, z = torch.empty_like(x), torch.empty_like(x)
    thff.ThunderFFT_rms_norm("half", x, weight, EPS, y, 40, cols)
    q, scales, _ = run8("half", x, None, weight, 128)
    x[7, cols // 2] = junk
    thff.ThunderFFT_rms_norm("half", x, weight, EPS, z, 40, cols)
    p, other, _ = run8("half", x, None, weight, 128)
    rest = [r for r in range(40) if r != 7]
    assert torch.equal(y[rest], z[rest]) and z[7].isnan().any()
    assert torch.equal(q.view(torch.uint8)[rest], p.view(torch.uint8)[rest]) and torch.equal(scales[rest], other[rest])
    assert p[7].float().isnan().any() and (junk != junk) == bool(p[7].float().isnan().all())


@pytest.mark.parametrize("T", list(oracle.TYPES))
@pytest.mark.parametrize("cols", [5, 64, 130, 777, 2048, 20011, 40001])
@pytest.mark.parametrize("large", [float("inf"), 3.0e38])
def test_8bit_infinite_scales(T, cols, large):
    """An infinite weight, or one whose product is out of range, makes its block's scale infinite: the finite
    values over it are 0, the infinite one a NaN, and other blocks are as without it."""
    x, residual, weight, *_ = values(23, T, 9, cols)
    at = cols // 2
    x[:, at], residual[:, at] = 64, 32
    for block in (128, cols):
        clean, fine, _ = run8(T, x, residual, weight, block)
        wild = weight.clone()
        wild[at] = large
        q, scales, _ = run8(T, x, residual, wild, block)
        hit = at // block
        assert (scales[:, hit] == float("inf")).all()
        inside = torch.arange(cols, device="cuda") // block == hit
        inside[at] = False
        assert (q.float()[:, inside] == 0).all() and q[:, at].float().isnan().all()
        outside = torch.arange(cols, device="cuda") // block != hit
        assert torch.equal(q.view(torch.uint8)[:, outside], clean.view(torch.uint8)[:, outside])
        rest = [b for b in range(scales.shape[1]) if b != hit]
        assert torch.equal(scales[:, rest], fine[:, rest])


def test_no_rows():
    """No rows: the weight's gradient is zeros, whatever the workspace."""
    dw = torch.full((40,), GUARD, device="cuda")
    thff.ThunderFFT_rms_norm_backward("half", 0, 0, 0, 0, 0, dw, 0, 0, 40)
    assert (dw == 0).all()
    thff.ThunderFFT_rms_norm("half", 0, 0, EPS, 0, 0, 40)
    thff.ThunderFFT_rms_norm_8bit("half", 0, 0, EPS, 0, 0, 0, 40)


@pytest.mark.parametrize("size", [(4099, 520), (700, 20011)], ids=str)
def test_same_bits_each_time(size):
    args = values(10, "bfloat16", *size)
    first = run("bfloat16", *args)
    for _ in range(3):
        again = run("bfloat16", *args)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_streams_and_graph_replays():
    """On a stream of its own, captured, and replayed with new inputs and eager calls between."""
    rows, cols = 3000, 520
    args = values(11, "bfloat16", rows, cols)
    x, residual, weight, dy, dsum = args
    y, total, dx, rstd, dw = (torch.empty_like(v) for v in (x, x, x, x[:, 0].float(), weight))
    q, scales = torch.empty(rows, cols, dtype=torch.uint8, device="cuda"), torch.empty(rows, 5, device="cuda")
    workspace = torch.empty(thff.rms_norm_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")

    def calls(stream):
        thff.ThunderFFT_rms_norm_async("bfloat16", x, weight, EPS, y, rows, cols, d_residual=residual, d_sum=total, d_rstd=rstd,
                                       stream=stream)
        thff.ThunderFFT_rms_norm_8bit_async("bfloat16", x, weight, EPS, q, scales, rows, cols, d_residual=residual, stream=stream)
        thff.ThunderFFT_rms_norm_backward_async("bfloat16", dy, total, rstd, weight, dx, dw, workspace, rows, cols, d_dsum=dsum,
                                                stream=stream)

    def check(new):
        want = run("bfloat16", *new)
        for name, v in (("y", y), ("sum", total), ("dx", dx), ("dweight", dw), ("rstd", rstd)):
            assert torch.equal(want[name], v), name
        want = run8("bfloat16", *new[:3], 128)
        assert torch.equal(want[0].view(torch.uint8), q) and torch.equal(want[1], scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls(side)
    torch.cuda.synchronize()
    check(args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for k in range(4):
        new = values(50 + k, "bfloat16", rows, cols)
        for old, v in zip(args, new):
            old.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check(new)


@pytest.mark.parametrize("shape", [(40,), (3, 5, 72), (2, 3, 4, 16), (4, 0, 8)], ids=str)
def test_tensor_functions(shape):
    gen = torch.Generator().manual_seed(12)
    x, residual, dy, dsum = (torch.randn(*shape, generator=gen).to(torch.bfloat16).cuda() for _ in range(4))
    weight = torch.randn(shape[-1], generator=gen).cuda()
    leaves = [v.requires_grad_() for v in (x, weight, residual)]
    y, total = thff.rms_norm(*leaves)
    torch.autograd.backward([y, total], [dy, dsum])
    flat = [v.detach().reshape(-1, shape[-1]) for v in (x, residual, dy, dsum)]
    want = oracle.rms("bfloat16", flat[0], weight, EPS, flat[1], flat[2], flat[3])
    got = dict(y=y, sum=total, dx=x.grad, dweight=weight.grad)
    for name in want:
        oracle.check(name, got[name].reshape(want[name][0].shape), want[name])
    assert torch.equal(x.grad, residual.grad)
    # Without a residual, and the sums alone.
    for v in leaves:
        v.grad = None
    y = thff.rms_norm(x, weight)
    y.backward(dy)
    want = oracle.rms("bfloat16", flat[0], weight, EPS, None, flat[2])
    for name, v in (("y", y), ("dx", x.grad), ("dweight", weight.grad)):
        oracle.check(name, v.reshape(want[name][0].shape), want[name])
    x.grad = None
    thff.rms_norm(x, None, residual)[1].backward(dsum)
    assert torch.equal(x.grad, dsum)
    for block in (128, None):
        q, scales, total = thff.rms_norm_8bit(x, weight, residual, block=block)
        assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scales.shape == (*shape[:-1], 1)
        assert len(thff.rms_norm_8bit(x, weight)) == 2
    with pytest.raises(ValueError, match="block"):
        thff.rms_norm_8bit(x, block=64)
    with pytest.raises(ValueError, match="residual"):
        thff.rms_norm(x, None, x.float())
