"""Definitions in 64 bits of the layer norm, gated recurrence and gated linear
unit, with bounds on what their kernels may be off by.

A kernel computes in fp32 and rounds its results once. With u = 2^-24 (half a
step of fp32) and `half` half a step of the result's type, every bound is

    half |result| + u * (the absolute terms of the result, each times the number
                         of fp32 roundings that it goes through)

and, where an intermediate is rounded to the type as well, half of it carried
through the formula. Sigmoids count 8 roundings for exp2, add, reciprocal and
product (each instruction within one step) and 2 |x| for the argument's.
"""

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def leaf(t):
    return None if t is None else t.detach().double().cpu().requires_grad_(True)


def sig(x):
    return torch.sigmoid(x)


def silu_slope(x):
    return sig(x) * (1 + x * sig(-x))


# ------------------------------------------------------------------ layer norm
SUM = 64  # additions that a value goes through in a sum over a row (lane, wave, block)


def norm_oracle(x, w, b, r, dy, ds, eps=1e-5):
    """[(exact, bound)] for y, s, dx, dw, db (s where r is given; db where b is)."""
    dt = x.dtype
    h = half(dt)
    x, w, b, r = leaf(x), leaf(w), leaf(b), leaf(r)
    dy, ds = dy.double().cpu(), None if ds is None else ds.double().cpu()
    s = x if r is None else x + r
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((s - mean).square().mean(-1, keepdim=True) + eps)
    n = (s - mean) * rstd
    y = n * w + (0 if b is None else b)
    outs, seeds = ([y], [dy]) if r is None else ([y, s], [dy, ds])
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(outs, leaves, seeds)
    with torch.no_grad():
        # n: the mean's error, then a few roundings of its own; the variance's
        # relative error is SUM / 2 roundings of rstd at most
        size = s.abs() if r is None else x.abs() + r.abs()
        en = U * (SUM * size.mean(-1, keepdim=True) * rstd + 4 * size * rstd + (SUM + 8) * n.abs())
        er = (SUM + 8) * U + 0 * rstd  # of rstd, relative
        ey = en * w.abs() + 4 * U * (y.abs() + (n * w).abs()) + h * y.abs()
        res = [(y.detach(), ey)]
        if r is not None:
            res.append((s.detach(), (h + 2 * U) * s.abs()))
        g = dy * w
        gn, eg = (g * n).mean(-1, keepdim=True), 2 * U * g.abs()
        egn = (g.abs() * en + eg * n.abs() + SUM * U * (g * n).abs()).mean(-1, keepdim=True)
        edx = rstd * (eg + SUM * U * g.abs().mean(-1, keepdim=True) + en * gn.abs() + (n.abs() + en) * egn
                      + er * (g.abs() + g.abs().mean(-1, keepdim=True) + (n * gn).abs()))
        dx = grads[0]
        edx = edx + 2 * U * (0 if ds is None else ds.abs()) + h * dx.abs()
        flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
        rows = 64 + flat(dy).shape[0] / 512  # additions down a column
        dw = grads[1]
        edw = flat(dy.abs() * en + rows * U * (dy * n).abs()).sum(0) + h * dw.abs()
        res += [(dx, edx), (dw, edw)]
        if b is not None:
            res.append((grads[2], rows * U * flat(dy).abs().sum(0) + h * grads[2].abs()))
    return res


# ------------------------------------------------------------ gated recurrence
STEP = 16  # roundings of a step's two terms: a sigmoid, its product, the scan's joins


def recurrence_oracle(gates, h0, lengths, dy, dhT):
    """[(exact, bound)] for y, hT, dgates, dh0."""
    dt = gates.dtype
    h = half(dt)
    T, B, H3 = gates.shape
    H = H3 // 3
    f, v, o = gates.detach().double().cpu().unflatten(-1, (3, H)).unbind(2)
    state = torch.zeros(B, H).double() if h0 is None else h0.detach().double().cpu()
    dy = torch.zeros(T, B, H).double() if dy is None else dy.double().cpu()
    R = torch.zeros(B, H).double() if dhT is None else dhT.double().cpu()
    real = torch.ones(T, B, 1, dtype=torch.bool)
    if lengths is not None:
        real = (torch.arange(T)[:, None] < lengths.cpu()[None, :]).unsqueeze(-1)
    zero = torch.zeros(1).double()
    f, v, o, dy = (torch.where(real, t, zero) for t in (f, v, o, dy))  # whatever a pad holds
    a, keep = torch.where(real, sig(f), zero + 1), torch.where(real, sig(-f), zero)
    ef, eo = (STEP + 2 * f.abs()) * U, (STEP + 2 * o.abs()) * U
    silu, slope = o * sig(o), silu_slope(o)
    eslope = eo * (sig(o) * (1 + o.abs()))
    y, ey = torch.zeros_like(dy), torch.zeros_like(dy)
    before, ebefore = torch.zeros_like(dy), torch.zeros_like(dy)
    after, eafter = torch.zeros_like(dy), torch.zeros_like(dy)
    size, err = state.abs(), torch.zeros_like(state)
    for t in range(T):
        before[t], ebefore[t] = state, err
        err = a[t] * err + ef[t] * (a[t] * size + (keep[t] * v[t]).abs())
        size = a[t] * size + (keep[t] * v[t]).abs()
        state = a[t] * state + keep[t] * v[t]
        after[t], eafter[t] = state, err
        y[t] = state * silu[t]
        ey[t] = silu[t].abs() * err + (eo[t] + h) * y[t].abs()
    hT, ehT = state, err
    p = dy * silu
    dgates, edg = torch.zeros_like(torch.cat([f, v, o], -1)), torch.zeros(T, B, H3).double()
    size, err = R.abs(), torch.zeros_like(R)
    for t in reversed(range(T)):
        G, eG, Gs = R + p[t], err + eo[t] * p[t].abs() + 2 * U * size, size + p[t].abs()
        d = before[t] - v[t]
        df, dv, do = G * d * a[t] * keep[t], G * keep[t], dy[t] * after[t] * slope[t]
        edf = (eG * d.abs() + G.abs() * (ebefore[t] + 2 * U * (before[t].abs() + v[t].abs()))) * a[t] * keep[t]
        edf = edf + (2 * ef[t] + h) * df.abs()
        edv = eG * keep[t] + (ef[t] + h) * dv.abs()
        edo = dy[t].abs() * (slope[t].abs() * eafter[t] + eslope[t] * after[t].abs()) + (4 * U + h) * do.abs()
        dgates[t], edg[t] = torch.cat([df, dv, do], -1), torch.cat([edf, edv, edo], -1)
        R, err, size = a[t] * G, a[t] * eG + ef[t] * a[t] * Gs, a[t] * Gs
    return [(y, ey), (hT, ehT + U * hT.abs()), (dgates, edg), (R, err + U * R.abs())]


# ----------------------------------------------------------- gated linear unit
def linear_oracle(x, w, b, dy, device="cpu"):
    """[(exact, bound)] for y, dx, dw, db (db where b is given), computed on `device`."""
    dt = x.dtype
    h = half(dt)
    K, F = x.shape[-1], w.shape[0] // 2
    shape = x.shape
    M = shape[:-1].numel()
    x, w = x.detach().to(device).double().reshape(M, K), w.detach().to(device).double()
    dy = dy.to(device).double().reshape(M, F)
    p, ep = x @ w.t(), (K + 4) * U * (x.abs() @ w.abs().t())
    if b is not None:
        bias = b.detach().to(device).double()
        p, ep = p + bias, ep + 2 * U * (bias.abs() + p.abs())
    g, u = p[:, :F], p[:, F:]
    eg, eu = ep[:, :F], ep[:, F:]
    silu, slope, es = g * sig(g), silu_slope(g), (STEP + 2 * g.abs()) * U
    y = silu * u
    # |silu'| <= 1.1 and |silu''| <= 0.5 everywhere
    ey = 1.1 * eg * u.abs() + silu.abs() * eu + (es + h) * y.abs()
    dg, du = dy * u * slope, dy * silu
    edg = dy.abs() * (0.5 * eg * u.abs() + 1.1 * eu + es * u.abs() * sig(g) * (1 + g.abs()))
    edu = dy.abs() * (1.1 * eg + es * silu.abs())
    dp, edp = torch.cat([dg, du], -1), torch.cat([edg, edu], -1)
    edb = edp + 64 * U * dp.abs() + M * U * dp.abs()
    edp = edp + (h + U) * dp.abs()  # dp is rounded to the type for the next products
    dx, dw = dp @ w, dp.t() @ x
    edx = edp @ w.abs() + (2 * F + 4) * U * (dp.abs() @ w.abs()) + h * dx.abs()
    edw = edp.t() @ x.abs() + (M + 64) * U * (dp.abs().t() @ x.abs()) + h * dw.abs()
    res = [(y.reshape(*shape[:-1], F), ey.reshape(*shape[:-1], F)),
           (dx.reshape(shape), edx.reshape(shape)), (dw, edw)]
    if b is not None:
        res.append((dp.sum(0), edb.sum(0) + h * dp.sum(0).abs()))
    return [(exact.cpu(), bound.cpu()) for exact, bound in res]


# Smallest step of fp32 and bf16 alike: results below it flush to zero.
TINY = 2.0 ** -126


def check(name, got, want):
    """Each value within its bound; nothing may be non-finite where the exact one is finite."""
    exact, bound = want
    assert got.shape == exact.shape, f"{name}: {tuple(got.shape)} != {tuple(exact.shape)}"
    if not got.numel():
        return
    off = (got.detach().double().cpu() - exact).abs()
    bad = ~(off <= bound + TINY)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((off / (bound + TINY)).max()):.3g} times its bound at "
                           f"{int((off / (bound + TINY)).argmax())}")
