"""The sequence operators in 64 bits on the CPU, step by step from their definitions, and
how far results computed in 32 bits may be from them.

The bounds follow the roundings of the formulas, with u = 2^-24:
  gate   e = exp(-|g|) through exp2: the exponent is off by 2 u |g| log2(e) (product and
         constant), exp2 by 2 u; 1 + e and e r by u each, the reciprocal by 2 u.  f and
         1 - f are off by (2 |g| + 8) u of their size at most.
  scan   a step multiplies by f, adds (1 - f) x and rounds; M is the recurrence of the
         sizes |x|, |state|, which no partial result exceeds in whichever order steps are
         joined, and joining rounds each term at most twice as often.
  norm   sums over c values by lanes that add at most c / 64 terms one after the other, then
         in trees: off by (c / 64 + 16) u of the sum of sizes.  Sums over r rows:
         (r / 32 + 64) u.
An output in T adds half a unit of its last place (of the least normal's at least).
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
TYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
_ROUND = {"float": (2.0 ** -24, 2.0 ** -149), "half": (2.0 ** -11, 2.0 ** -25),
          "bfloat16": (2.0 ** -8, 2.0 ** -134)}


def rounding(T, value, error):
    """error with that of storing value +- error in T."""
    rel, least = _ROUND[T]
    return error + (value.abs() + error) * rel + least


def _steps(v, layout):
    """(n, batch, channels) in 64 bits."""
    v = v.detach().cpu().double()
    return v.permute(1, 0, 2) if layout == "channels_last" else v.permute(2, 0, 1)


def _back(v, layout):
    return v.permute(1, 0, 2) if layout == "channels_last" else v.permute(1, 2, 0)


def scan(T, layout, x, gate, state=None, lengths=None, dy=None, dstate=None):
    """{name: (value, bound)} of y, state and, with dy, dx, dgate and dstate."""
    x, gate = _steps(x, layout).clone(), _steps(gate, layout).clone()
    n, batch, channels = x.shape
    inside = torch.ones(n, batch, 1, dtype=torch.bool)
    if lengths is not None:
        inside = (torch.arange(n).unsqueeze(1) < lengths.cpu()).unsqueeze(2)
    x[~inside.expand_as(x)] = 0.0
    gate[~inside.expand_as(gate)] = 0.0
    f, s = torch.sigmoid(gate), torch.sigmoid(-gate)
    g = (2 * gate.abs() + 8) * U  # relative error of either
    h = torch.zeros(batch, channels, dtype=torch.float64) if state is None else state.cpu().double()
    M, E = h.abs(), torch.zeros_like(h)
    before, before_M, before_E, hs, Es = [], [], [], [], []
    for t in range(n):
        on = inside[t]
        before.append(h), before_M.append(M), before_E.append(E)
        new = f[t] * h + s[t] * x[t]
        new_M = f[t] * M + s[t] * x[t].abs()
        new_E = f[t] * E + 2 * ((g[t] + 2 * U) * new_M + 2 * U * new_M)
        h, M, E = torch.where(on, new, h), torch.where(on, new_M, M), torch.where(on, new_E, E)
        hs.append(torch.where(on, new, 0.0)), Es.append(torch.where(on, new_E, 0.0))

    def laid(values):
        return _back(torch.stack(values) if n else torch.zeros(0, batch, channels, dtype=torch.float64),
                     layout)

    y = laid(hs)
    got = {"y": (y, rounding(T, y, laid(Es))), "state": (h, rounding("float", h, E))}
    if dy is None:
        return got
    dy = _steps(dy, layout).clone()
    dy[~inside.expand_as(dy)] = 0.0
    c = torch.zeros(batch, channels, dtype=torch.float64) if dstate is None else dstate.cpu().double()
    C, CE = c.abs(), torch.zeros_like(c)
    dxs, dxe, dgs, dge = [None] * n, [None] * n, [None] * n, [None] * n
    for t in range(n - 1, -1, -1):
        on = inside[t]
        lam, L = dy[t] + c, dy[t].abs() + C
        LE = CE + 4 * U * L
        D, DE = before[t] - x[t], before_E[t]
        DM = before_M[t] + x[t].abs()
        fs = f[t] * s[t]
        dxs[t] = torch.where(on, s[t] * lam, 0.0)
        dxe[t] = torch.where(on, s[t] * (LE + (g[t] + 2 * U) * L), 0.0)
        dgs[t] = torch.where(on, lam * D * fs, 0.0)
        dge[t] = torch.where(on, fs * (LE * DM + L * (DE + 2 * U * DM) + L * DM * (2 * g[t] + 6 * U)), 0.0)
        new, new_C = f[t] * lam, f[t] * L
        new_CE = f[t] * LE + 2 * (g[t] + 2 * U) * new_C
        c, C, CE = torch.where(on, new, c), torch.where(on, new_C, C), torch.where(on, new_CE, CE)
    dx, dgate = laid(dxs), laid(dgs)
    got["dx"] = (dx, rounding(T, dx, laid(dxe)))
    got["dgate"] = (dgate, rounding(T, dgate, laid(dge)))
    got["dstate"] = (c, rounding("float", c, CE))
    return got


def norm(T, x, weight, bias, eps, dy=None):
    """{name: (value, bound)} of y and, with dy, dx, dweight and dbias."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    w = torch.ones(cols, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    b = torch.zeros(cols, dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    k = (cols / 64 + 16) * U
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    size = x.abs().mean(1, keepdim=True)
    off = k * size  # of the mean
    xh = (x - mean) * rstd
    # rstd: half the relative error of var + eps (its sum, and the mean's error squared), and
    # the root and the reciprocal.
    r = 0.5 * (k + 4 * U + (off * rstd) ** 2) + 4 * U
    xe = rstd * (off + 2 * U * (x.abs() + mean.abs())) + xh.abs() * (r + 2 * U)
    y = xh * w + b
    got = {"y": (y, rounding(T, y, w.abs() * xe + 2 * U * ((w * xh).abs() + b.abs())))}
    if dy is None:
        return got
    dy = dy.detach().cpu().double()
    g = dy * w
    mg, al = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    mge = k * g.abs().mean(1, keepdim=True)
    ale = (k + 4 * U) * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * xe).mean(1, keepdim=True)
    dx = rstd * (g - mg - xh * al)
    parts = g.abs() + mg.abs() + (xh * al).abs()
    dxe = rstd * (4 * U * parts + mge + xh.abs() * ale + xe * al.abs()) + rstd * parts * (r + 2 * U)
    got["dx"] = (dx, rounding(T, dx, dxe))
    q = (rows / 32 + 64) * U
    dw = (dy * xh).sum(0)
    got["dweight"] = (dw, rounding("float", dw, (q + 4 * U) * (dy * xh).abs().sum(0) + (dy.abs() * xe).sum(0)))
    db = dy.sum(0)
    got["dbias"] = (db, rounding("float", db, q * dy.abs().sum(0)))
    return got


def check(name, got, expected):
    """got within its bound of the oracle's value, everywhere."""
    value, bound = expected
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), name
    over = (got - value).abs() - bound
    if over.numel():
        worst = int(over.argmax())
        assert float(over.max()) <= 0, (
            f"{name}: {float(got.flatten()[worst])} instead of {float(value.flatten()[worst])} "
            f"(bound {float(bound.flatten()[worst]):.3g}) at {worst}, {int((over > 0).sum())} values off")
