"""A state space block's operators in 64 bits on the CPU, from their definitions, and how far
results computed in 32 bits may be from them.

Values come with bounds, which follow the roundings of the formulas with u = 2^-24; exp, the
reciprocal and the square root are off by 2 u, and what is below 2^-126 may be lost:
  exp(v)     through exp2: the exponent is off by 2 u of its size more (constant and product).
  sigmoid    (2 |v| + 8) u of itself: exp, a sum, a reciprocal.
  softplus   of v = delta + bias, off by u |v|: the slope carries that; exp(-|v|), the logarithm of
             the rounded 1 + exp(-|v|), what that rounding lost, and a sum: (1.25 |v| + 11) u of
             log(1 + exp(-|v|)) and u of itself (the test of step sizes has the terms and holds the
             kernels to them), taken as (2 |v| + 16) u of itself.
  conv       width products, added one after the other: (width + 1) u of the sum of sizes.
  scan       a step multiplies by exp(dt a) and adds dt x b; M is the recurrence of the sizes.
             Segments join by exp(a sum of dt), whose sum is off by no more than the steps' roundings
             are together: every step's are counted twice.
  norm       as the layer norm's sums: (cols / 64 + 16) u of the sum of sizes.
  sums over steps and channels: lanes and waves add at most `count` / 4 terms one after the other,
             or 80, whichever is more, then trees: (count / 4 + 80) u of the sum of sizes.
An output in T adds half a unit of its last place (of the least normal's at least).
"""
from __future__ import annotations

import torch

from sequence_oracle import TYPES, U, check, rounding  # noqa: F401

TINY = 2.0 ** -126
D = torch.float64


def _d(v):
    return None if v is None else v.detach().cpu().double()


def _inside(lengths, batch, n):
    """(batch, n, 1): whether a step is before its sequence's end; and the ends."""
    ends = torch.full((batch,), n) if lengths is None else lengths.cpu().long().clamp(0, n)
    return (torch.arange(n) < ends.unsqueeze(1)).unsqueeze(2), ends


def _sigmoid(v, e):
    """1 / (1 + exp(-v)) of v off by e."""
    f = torch.sigmoid(v)
    return f, f * (1 - f) * e + f * (2 * v.abs() + 8) * U + TINY


def _silu(v, e):
    f, fe = _sigmoid(v, e)
    # The slope is below 1.1, and steeper than 0.6 of the error nowhere.
    return v * f, 1.1 * e + v.abs() * (f * (2 * v.abs() + 8) * U) + 2 * U * (v * f).abs() + TINY * (1 + v.abs())


def _silu_slope(v, e):
    f, fe = _sigmoid(v, torch.zeros_like(e))
    slope = f * (1 + v * (1 - f))
    return slope, 0.5 * e + fe * (1 + 2 * v.abs()) + 4 * U * (f + (v * f * (1 - f)).abs())


def conv(T, x, weight, bias, state=None, lengths=None, silu=True, dy=None, dstate=None):
    """{name: (value, bound)} of y and state and, with dy, dx, dweight, dbias and dstate."""
    x, w = _d(x), _d(weight)
    batch, n, channels = x.shape
    width = w.shape[1]
    inside, ends = _inside(lengths, batch, n)
    xe = torch.cat([torch.zeros(batch, width - 1, channels, dtype=D) if state is None else _d(state),
                    torch.where(inside, x, 0.0)], 1)
    b = torch.zeros(channels, dtype=D) if bias is None else _d(bias)
    p, size = b.expand(batch, n, channels).clone(), b.abs().expand(batch, n, channels).clone()
    for k in range(width):
        p += w[:, k] * xe[:, k:k + n]
        size += (w[:, k] * xe[:, k:k + n]).abs()
    pe = (width + 1) * U * size
    y, ye = _silu(p, pe) if silu else (p, pe)
    y, ye = torch.where(inside, y, 0.0), torch.where(inside, ye, 0.0)
    at = (ends.unsqueeze(1) + torch.arange(width - 1)).unsqueeze(2).expand(-1, -1, channels)
    last = xe.gather(1, at)
    got = {"y": (y, rounding(T, y, ye)), "state": (last, torch.zeros_like(last))}
    if dy is None:
        return got
    slope, se = _silu_slope(p, pe) if silu else (torch.ones_like(p), torch.zeros_like(p))
    dy = torch.where(inside, _d(dy), 0.0)
    dp, de = dy * slope, dy.abs() * (se + 2 * U * slope.abs())
    dxe, dxee = torch.zeros_like(xe), torch.zeros_like(xe)
    sizes = torch.zeros_like(xe)
    if dstate is not None:
        dxe.scatter_(1, at, _d(dstate))
        sizes.scatter_(1, at, _d(dstate).abs())
    dw, dwe = torch.zeros_like(w), torch.zeros_like(w)
    count = (batch * n / 4 + 80) * U
    for k in range(width):
        dxe[:, k:k + n] += w[:, k] * dp
        sizes[:, k:k + n] += (w[:, k] * dp).abs()
        dxee[:, k:k + n] += w[:, k].abs() * de
        term = dp * xe[:, k:k + n]
        dw[:, k] = term.sum((0, 1))
        dwe[:, k] = count * term.abs().sum((0, 1)) + (de * xe[:, k:k + n].abs()).sum((0, 1))
    dxee += (width + 1) * U * sizes
    dx, dxe_bound = torch.where(inside, dxe[:, width - 1:], 0.0), torch.where(inside, dxee[:, width - 1:], 0.0)
    got["dx"] = (dx, rounding(T, dx, dxe_bound))
    got["dstate"] = (dxe[:, :width - 1], rounding(T, dxe[:, :width - 1], dxee[:, :width - 1]))
    got["dweight"] = (dw, rounding("float", dw, dwe))
    db = dp.sum((0, 1))
    got["dbias"] = (db, rounding("float", db, count * dp.abs().sum((0, 1)) + de.sum((0, 1))))
    return got


def state(T, x, delta, a, b, c, skip=None, gate=None, delta_bias=None, state=None, lengths=None, dy=None, dstate=None):
    """{name: (value, bound)} of y and state and, with dy, of the gradients.  b and c: (batch, n, groups, order)."""
    x, delta, a, b, c = (_d(v) for v in (x, delta, a, b, c))
    batch, n, channels = x.shape
    groups, order = b.shape[2:]
    inside, ends = _inside(lengths, batch, n)

    def at_steps(v):
        return torch.where(inside, v, 0.0)

    def shared(v):
        """(batch, n, channels, order)"""
        v = torch.where(inside.unsqueeze(3), v, 0.0)
        return v.unsqueeze(3).expand(-1, -1, -1, channels // groups, -1).reshape(batch, n, channels, order)

    x, b, c = at_steps(x), shared(b), shared(c)
    zeros = torch.zeros(channels, dtype=D)
    skip, delta_bias = (zeros if v is None else _d(v) for v in (skip, delta_bias))
    raw = delta + delta_bias
    soft = torch.where(inside, raw, 0.0)
    opened, opened_e = _sigmoid(soft, U * soft.abs())
    dt = at_steps(torch.clamp(soft, min=0.0) + torch.log1p(torch.exp(-soft.abs())))
    dte = at_steps(opened * U * soft.abs() + dt * (2 * soft.abs() + 16) * U + TINY)
    u = dt * x
    ue = dte * x.abs() + U * u.abs()
    exponent = dt.unsqueeze(3) * a
    keep = torch.exp(exponent)
    # Relative to keep.
    keep_e = dte.unsqueeze(3) * a.abs() + 3 * U * exponent.abs() + 2 * U
    keep_e = torch.where(inside.unsqueeze(3), keep_e, 0.0)
    enter, enter_e = u.unsqueeze(3) * b, ue.unsqueeze(3) * b.abs() + U * (u.unsqueeze(3) * b).abs()
    h = torch.zeros(batch, channels, order, dtype=D) if state is None else _d(state)
    M, E = h.abs(), torch.zeros_like(h)
    hs, Ms, Es = [h], [M], [E]
    on = inside.unsqueeze(3)
    for t in range(n):
        h = keep[:, t] * h + enter[:, t]
        E = keep[:, t] * E + 2 * (keep_e[:, t] + 2 * U * on[:, t]) * keep[:, t] * M + enter_e[:, t] + TINY * on[:, t]
        M = keep[:, t] * M + enter[:, t].abs()
        E = E + 2 * U * M * on[:, t]
        hs.append(h), Ms.append(M), Es.append(E)
    hs, Ms, Es = (torch.stack(v, 1) for v in (hs, Ms, Es))
    before, new = slice(0, n), slice(1, n + 1)
    inner = (c * hs[:, new]).sum(3) + skip * x
    inner_e = ((c.abs() * Es[:, new]).sum(3) + (order + 4) * U * ((c.abs() * Ms[:, new]).sum(3) + (skip * x).abs()))
    z, ze = (torch.ones_like(x), torch.zeros_like(x)) if gate is None else _silu(_d(gate), torch.zeros_like(x))
    gv = None if gate is None else _d(gate)
    y = at_steps(inner * z)
    ye = at_steps(inner_e * z.abs() + inner.abs() * ze + 2 * U * (inner * z).abs())
    got = {"y": (y, rounding(T, y, ye)), "state": (hs[:, n], rounding("float", hs[:, n], Es[:, n]))}
    if dy is None:
        return got
    dy = at_steps(_d(dy))
    dn = dy * z
    dne = dy.abs() * ze + 2 * U * dn.abs()
    if gate is not None:
        slope, slope_e = _silu_slope(gv, torch.zeros_like(gv))
        dg = at_steps(dy * inner * slope)
        got["dgate"] = (dg, rounding(T, dg, at_steps(dy.abs() * (inner_e * slope.abs() + inner.abs() * slope_e) + 3 * U * dg.abs())))
    lam = torch.zeros(batch, channels, order, dtype=D) if dstate is None else _d(dstate)
    L, LE = lam.abs(), torch.zeros_like(lam)
    lams, Ls, LEs = [None] * n, [None] * n, [None] * n
    for t in range(n - 1, -1, -1):
        add = dn[:, t].unsqueeze(2) * c[:, t]
        lam, L = lam + add, L + add.abs()
        LE = LE + dne[:, t].unsqueeze(2) * c[:, t].abs() + 4 * U * L * on[:, t]
        lams[t], Ls[t], LEs[t] = lam, L, LE
        LE = keep[:, t] * LE + 2 * (keep_e[:, t] + 2 * U * on[:, t]) * keep[:, t] * L + TINY * on[:, t]
        lam, L = keep[:, t] * lam, keep[:, t] * L
    got["dstate"] = (lam, rounding("float", lam, LE))
    if n == 0:
        lams, Ls, LEs = (torch.zeros(batch, 0, channels, order, dtype=D) for _ in range(3))
    else:
        lams, Ls, LEs = (torch.stack(v, 1) for v in (lams, Ls, LEs))
    order_u = (order + 4) * U
    du = (lams * b).sum(3)
    due = (LEs * b.abs()).sum(3) + order_u * (Ls * b.abs()).sum(3)
    q = lams * keep * hs[:, before]
    size = Ls * keep * Ms[:, before]
    qe = keep * (LEs * Ms[:, before] + Ls * Es[:, before]) + size * (keep_e + 4 * U)
    de = (q * a).sum(3)
    dee = (qe * a.abs()).sum(3) + order_u * (size * a.abs()).sum(3)
    dx = at_steps(du * dt + dn * skip)
    dxe = at_steps(due * dt + du.abs() * dte + dne * skip.abs() + 3 * U * ((Ls * b.abs()).sum(3) * dt + (dn * skip).abs()))
    got["dx"] = (dx, rounding(T, dx, dxe))
    dr = at_steps((du * x + de) * opened)
    parts = (Ls * b.abs()).sum(3) * x.abs() + (size * a.abs()).sum(3)
    dre = at_steps((due * x.abs() + dee + 4 * U * parts) * opened + parts * opened_e)
    got["ddelta"] = (dr, rounding(T, dr, dre))
    count = (batch * n / 4 + 80) * U
    value, sizes, off = dr.sum((0, 1)), at_steps(parts * opened).sum((0, 1)), dre.sum((0, 1))
    got["ddelta_bias"] = (value, rounding("float", value, count * sizes + off))
    value = (dn * x).sum((0, 1))
    got["dskip"] = (value, rounding("float", value, count * (dn * x).abs().sum((0, 1)) + (dne * x.abs()).sum((0, 1))))
    d = dt.unsqueeze(3)
    value = (q * d).sum((0, 1))
    got["da"] = (value, rounding("float", value, count * (size * d).sum((0, 1)) + (qe * d + size * dte.unsqueeze(3)).sum((0, 1))))
    many = (channels // groups / 4 + 80) * U

    def of_group(v):
        return v.view(batch, n, groups, channels // groups, order).sum(3)

    w = u.unsqueeze(3)
    value = of_group(lams * w)
    got["db"] = (value, rounding(T, value, of_group(many * Ls * w.abs() + LEs * w.abs() + Ls * ue.unsqueeze(3))))
    w = dn.unsqueeze(3)
    value = of_group(hs[:, new] * w)
    got["dc"] = (value, rounding(T, value, of_group(many * Ms[:, new] * w.abs() + Es[:, new] * w.abs() + Ms[:, new] * dne.unsqueeze(3))))
    return got


def rms(T, x, weight, eps, residual=None, dy=None, dsum=None):
    """{name: (value, bound)} of y and sum and, with dy, dx and dweight."""
    s = x.detach().cpu()
    if residual is not None:
        # One rounding to T, which the 32-bit sum of two values of T does not change.
        s = (s.double() + residual.detach().cpu().double()).to(s.dtype)
    v = s.double()
    rows, cols = v.shape
    w = torch.ones(cols, dtype=D) if weight is None else _d(weight)
    k = (cols / 64 + 16) * U
    rstd = 1 / (v.square().mean(1, keepdim=True) + eps).sqrt()
    r = 0.5 * (k + 4 * U) + 4 * U  # of itself
    xh = v * rstd
    xe = xh.abs() * (r + U)
    y = xh * w
    got = {"y": (y, rounding(T, y, xe * w.abs() + 2 * U * y.abs())), "sum": (v, torch.zeros_like(v))}
    if dy is None:
        return got
    dy = _d(dy)
    g = dy * w
    al = (g * xh).mean(1, keepdim=True)
    ale = (k + 4 * U) * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * xe).mean(1, keepdim=True)
    more = torch.zeros_like(v) if dsum is None else _d(dsum)
    dx = rstd * (g - xh * al) + more
    parts = g.abs() + (xh * al).abs()
    dxe = rstd * (4 * U * parts + xh.abs() * ale + xe * al.abs()) + rstd * parts * (r + 2 * U) + 2 * U * (rstd * parts + more.abs())
    got["dx"] = (dx, rounding(T, dx, dxe))
    q = (rows / 32 + 64) * U
    dw = (dy * xh).sum(0)
    got["dweight"] = (dw, rounding("float", dw, (q + 4 * U) * (dy * xh).abs().sum(0) + (dy.abs() * xe).sum(0)))
    return got


def rms_8bit(T, x, weight, eps, block, residual=None):
    """(scales and their bound, y and its bound): a q * scale is within half a step of y."""
    s = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    # y in 64 bits, with what 32 bits are off.
    y, bound = rms("float", s.float(), weight, eps)["y"]
    rows, cols = y.shape
    wide = torch.nn.functional.pad(y, (0, -cols % block)).view(rows, -1, block)
    off = torch.nn.functional.pad(bound, (0, -cols % block)).view(rows, -1, block)
    scales = (wide.abs().amax(2) / 448).clamp(min=2.0 ** -126)
    return (scales, off.amax(2) / 448 + 4 * U * scales), (y, bound)
