"""The gated linear recurrence and layer norm in float64, forward and backward,
with the error bounds that a float32 evaluation has against them.

The bounds count roundings: a float32 operation is off by 2^-24 relative at most,
ex2.approx by 2^-22, rcp.approx by 2^-23 (their documented errors), the argument of
the exponential by two roundings, and an output by half a step of its type.
"""

from __future__ import annotations

import torch

from serving_reference import U, half_step, row_of, rounded, sequences

EX2, RCP = 2.0**-22, 2.0**-23
LEVELS = 16  # roundings that joining partial results adds to a value besides those of its own steps
TINY = 2.0**-120  # products of many gates leave float32's range


def gate(f, bound):
    """a, 1 - a and their relative bounds, and sigmoid(f), sigmoid(-f) with theirs."""
    f = f.double()
    low = torch.zeros((), dtype=torch.float64) if bound is None else bound.double()
    keep, take = torch.sigmoid(f), torch.sigmoid(-f)
    # t = exp(-|f|): the argument |f| log2 e is rounded twice. Behind |f| = 88 t is below 2^-126 or flushed to zero, and
    # what it adds or lacks is below TINY, so that infinite f have a bound too
    et = EX2 + 2 * U * f.abs().clamp(max=88) * 1.001 + 2 * U
    t = torch.exp(-f.abs())
    er = RCP + U + t / (1 + t) * et  # r = 1 / (1 + t)
    es = er + et + U  # t r
    ek, ee = torch.where(f >= 0, er, es), torch.where(f >= 0, es, er)
    # 1 - low is rounded, its products with keep and with take (or with r and then with t) are, and the sum is
    a = low + (1 - low) * keep
    ea = ((1 - low) * keep * (ek + 2 * U)) / a.clamp(min=1e-300) + U
    return dict(a=a, u=(1 - low) * take, ea=ea, eu=ee + 3 * U, keep=keep, take=take, ek=ek, et=ee + U)


def recurrence(x, f, bound=None, state=None, cu=None, slots=None, live=None, out=None, final=None):
    """Returns (y, bound of y, final states, bound of the final states). `out` and `final` are what the results hold
    where nothing is written."""
    dtype = x.dtype
    batch, seqlen, dim = x.shape
    xx = x.double().reshape(-1, dim)
    g = {k: v.expand(batch * seqlen, dim) for k, v in gate(f.reshape(-1, dim), bound).items()}
    y = torch.zeros_like(xx) if out is None else out.double().reshape(-1, dim).clone()
    yb = torch.zeros_like(y)
    segs = sequences(batch, seqlen, cu)
    if final is None:
        final = torch.zeros((len(segs), dim)) if state is None or slots is None else state
    final = final.double().clone()
    fb = torch.zeros_like(final)
    for i, (s, e) in enumerate(segs):
        row = row_of(i, slots, final.shape[0])
        h = torch.zeros(dim, dtype=torch.float64)
        if state is not None and row is not None and (live is None or int(live[i])):
            h = state[row].double().clone()
        mag, err = h.abs(), torch.zeros_like(h)
        for t in range(s, e):
            a, u = g["a"][t], g["u"][t]
            b = u * xx[t]
            err = a * err + a * mag * (g["ea"][t] + U) + b.abs() * (g["eu"][t] + U)
            h = a * h + b
            mag = a * mag + b.abs()
            err = err + U * mag
            y[t], yb[t] = h, rounded(h, err + LEVELS * U * mag + TINY, dtype)
        if row is not None:
            final[row], fb[row] = h, err + LEVELS * U * mag + TINY
            if s == e:
                fb[row] = 0
    return y.reshape(x.shape), yb.reshape(x.shape), final, fb


def recurrence_grad(dy, x, f, y, bound=None, state=None, cu=None, dlast=None, dx=None, df=None):
    """Returns four (value, bound) pairs: dx, df, d_lower_bound, d_initial_state."""
    dtype = dy.dtype
    batch, seqlen, dim = x.shape
    flat = lambda v: v.double().reshape(-1, dim)  # noqa: E731
    D, X, Y = flat(dy), flat(x), flat(y)
    g = {k: v.expand(batch * seqlen, dim) for k, v in gate(f.reshape(-1, dim), bound).items()}
    dx = torch.zeros_like(X) if dx is None else flat(dx).clone()
    df = torch.zeros_like(X) if df is None else flat(df).clone()
    bx, bf = torch.zeros_like(X), torch.zeros_like(X)
    lb, lbmag, lberr = (torch.zeros(dim, dtype=torch.float64) for _ in range(3))
    segs = sequences(batch, seqlen, cu)
    d0 = torch.zeros(len(segs), dim, dtype=torch.float64)
    b0 = torch.zeros_like(d0)
    for i, (s, e) in enumerate(segs):
        c = torch.zeros(dim, dtype=torch.float64) if dlast is None else dlast[i].double().clone()
        mag, err = c.abs(), torch.zeros(dim, dtype=torch.float64)
        for t in reversed(range(s, e)):
            G = D[t] + c
            gmag = D[t].abs() + mag
            gerr = err + (LEVELS + 1) * U * gmag + TINY
            before = Y[t - 1] if t > s else (torch.zeros(dim, dtype=torch.float64) if state is None else state[i].double())
            diff = before - X[t]
            u, a, keep, take = (g[k][t] for k in ("u", "a", "keep", "take"))
            dx[t] = u * G
            bx[t] = rounded(dx[t], u * gerr * 1.0001 + dx[t].abs() * (g["eu"][t] + 2 * U) + TINY, dtype)
            da = G * diff
            daerr = diff.abs() * gerr * 1.0001 + da.abs() * 3 * U
            df[t] = da * u * keep
            bf[t] = rounded(df[t], daerr * u * keep + df[t].abs() * (g["eu"][t] + g["ek"][t] + 4 * U) + TINY, dtype)
            lb += da * take
            lberr += daerr * take + (da * take).abs() * (g["et"][t] + 2 * U)
            lbmag += (da * take).abs()
            err = a * (err + U * gmag) + a * gmag * (g["ea"][t] + U)
            c, mag = a * G, a * gmag
        d0[i], b0[i] = c, (err + LEVELS * U * mag + TINY if e > s else 0)
    # any order of summation: fewer roundings in a row than there are tokens, and the joins
    lberr = lberr * 1.0001 + (batch * seqlen + LEVELS) * U * lbmag
    shape = x.shape
    return ((dx.reshape(shape), bx.reshape(shape)), (df.reshape(shape), bf.reshape(shape)), (lb, lberr), (d0, b0))


def _chain(n):
    """Additions that one value of a sum over n goes through at most: a thread's own, then a tree."""
    return 48 + n // 256


def norm(x, weight=None, bias=None, residual=None, eps=1e-5, rms=False):
    """Returns (y, bound), (s, bound), (stats, bound)."""
    dtype, dim = x.dtype, x.shape[-1]
    s = x
    if residual is not None:
        s = (x.float() + residual.float()).to(dtype)  # one float32 sum, one rounding: nothing is left open
    v = s.double().reshape(-1, dim)
    K = _chain(dim)
    if rms:
        mean, em = torch.zeros(v.shape[0], 1, dtype=torch.float64), torch.zeros(v.shape[0], 1, dtype=torch.float64)
    else:
        mean = v.mean(1, keepdim=True)
        em = (K + 2) * U * v.abs().mean(1, keepdim=True)
    d = v - mean
    ed = em + U * d.abs() * (0 if rms else 1)
    var = (d * d).mean(1, keepdim=True)
    ev = (2 * d.abs() * ed + ed * ed).mean(1, keepdim=True) + (K + 3) * U * var
    low = (var - ev).clamp(min=0) + eps
    # the square root and the quotient are off by a few units in the last place
    rstd = 1 / torch.sqrt(var + eps)
    er = rstd * (4 * U) + 0.5 * (ev + U * (var + eps)) * low ** -1.5
    w = torch.ones(dim, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(dim, dtype=torch.float64) if bias is None else bias.double()
    z = d * rstd * w
    ez = (ed * (rstd + er) + d.abs() * er) * w.abs() + 3 * U * z.abs()
    y = z + b
    yb = rounded(y, ez + 2 * U * (z.abs() + b.abs()), dtype)
    stats = torch.cat([mean, rstd], 1).reshape(*x.shape[:-1], 2)
    sb = torch.cat([em, er], 1).reshape(*x.shape[:-1], 2)
    return (y.reshape(x.shape), yb.reshape(x.shape)), (s.double(), torch.zeros_like(s.double())), (stats, sb)


def norm_grad(dy, x, weight, stats, dres=None, rms=False):
    """Returns (dx, bound), (d_weight, bound), (d_bias, bound)."""
    dtype, dim = dy.dtype, x.shape[-1]
    D, X = dy.double().reshape(-1, dim), x.double().reshape(-1, dim)
    st = stats.double().reshape(-1, 2)
    mean, rstd = (torch.zeros_like(st[:, :1]) if rms else st[:, :1]), st[:, 1:]
    w = torch.ones(dim, dtype=torch.float64) if weight is None else weight.double()
    xhat = (X - mean) * rstd
    ex = 2 * U * xhat.abs()
    g = D * w
    K = _chain(dim)
    sx = (g * xhat).mean(1, keepdim=True)
    esx = (g.abs() * (ex + 2 * U * xhat.abs())).mean(1, keepdim=True) + (K + 2) * U * (g * xhat).abs().mean(1, keepdim=True)
    sg, esg = torch.zeros_like(sx), torch.zeros_like(sx)
    if not rms:
        sg = g.mean(1, keepdim=True)
        esg = U * g.abs().mean(1, keepdim=True) + (K + 2) * U * g.abs().mean(1, keepdim=True)
    mag = g.abs() + sg.abs() + (xhat * sx).abs()
    inner = g - sg - xhat * sx
    ei = 4 * U * mag + esg + xhat.abs() * esx + ex * (sx.abs() + esx)
    dx = rstd * inner
    edx = rstd * ei + 2 * U * dx.abs()
    if dres is not None:
        r = dres.double().reshape(-1, dim)
        dx = dx + r
        edx = edx + 2 * U * ((rstd * mag) + r.abs())
    rows = D.shape[0]
    dw = (D * xhat).sum(0)
    ew = (D.abs() * ex).sum(0) + (rows + LEVELS) * U * (D * xhat).abs().sum(0)
    eb = (rows + LEVELS) * U * D.abs().sum(0)
    return (dx.reshape(x.shape), rounded(dx, edx, dtype).reshape(x.shape)), (dw, ew), (D.sum(0), eb)


__all__ = ["gate", "recurrence", "recurrence_grad", "norm", "norm_grad", "half_step"]
