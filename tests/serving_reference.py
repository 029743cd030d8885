"""The serving operators' definitions in float64, with the error bound that a
float32 evaluation has against them.

Every function returns (value, bound) pairs. The bounds count roundings: a
float32 operation is off by 2^-24 relative at most, ex2.approx, the fast
reciprocal and the softplus series by 2^-21 (their documented few units in the
last place, with the argument's own rounding counted apart), and the output's
rounding by half a step of its type.
"""

from __future__ import annotations

import torch

U = 2.0**-24  # a float32 rounding
F = 2.0**-21  # a fast elementary function


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def silu(v, verr):
    """v sigmoid(v) and its bound. The slope is at most 1.1; exp(-v) is off by F plus |v| 2^-23 relative (argument),
    which moves the result by that times |v| e / (1 + e)^2 <= 0.45, and |v|^2 e / (1 + e)^2 <= 0.88."""
    y = v * torch.sigmoid(v)
    return y, 1.1 * verr + F * 0.45 + 2 * U * 0.88 + F * y.abs()


def rounded(y, err, dtype):
    """Bound after rounding to the output type (2^-25: half of float16's smallest step)."""
    return err + half_step(dtype) * (y.abs() + err) + (2.0**-25 if dtype == torch.float16 else 0.0)


def sequences(batch, seqlen, cu):
    if cu is None:
        return [(b * seqlen, (b + 1) * seqlen) for b in range(batch)]
    cu = [int(v) for v in cu]
    return list(zip(cu, cu[1:]))


def row_of(i, slots, rows):
    if slots is None:
        return i
    s = int(slots[i])
    return s if 0 <= s < rows else None


def conv(x, weight, bias=None, state=None, cu=None, slots=None, live=None, silu_=True, channels_last=False, out=None,
         final=None):
    """x as the operator takes it. `out` and `final` are what the result holds where nothing is written. Returns
    (y, bound of y, final states)."""
    dtype = x.dtype
    xt = (x if channels_last else x.transpose(1, 2)).double()
    batch, seqlen, dim = xt.shape
    xt = xt.reshape(-1, dim)
    tail = weight.shape[1] - 1
    y = torch.zeros_like(xt) if out is None else (out if channels_last else out.transpose(1, 2)).double().reshape(-1, dim).clone()
    bound = torch.zeros_like(y)
    segs = sequences(batch, seqlen, cu)
    if final is None:
        final = torch.zeros((len(segs), dim, tail), dtype=dtype) if state is None or slots is None else state
    final = final.clone()
    for i, (a, b) in enumerate(segs):
        row = row_of(i, slots, final.shape[0])
        start = torch.zeros((tail, dim), dtype=torch.float64)
        if state is not None and row is not None and (live is None or int(live[i])):
            start = state[row].double().t()
        ext = torch.cat([start, xt[a:b]])
        v = torch.zeros((b - a, dim), dtype=torch.float64) if bias is None else bias.double().expand(b - a, dim).clone()
        mag = v.abs()
        for k in range(tail + 1):
            term = ext[k:k + b - a] * weight[:, k].double()
            v = v + term
            mag = mag + term.abs()
        err = (tail + 2) * U * mag
        if silu_:
            v, err = silu(v, err)
        y[a:b] = v
        bound[a:b] = rounded(v, err, dtype)
        if row is not None:
            final[row] = ext[ext.shape[0] - tail:].t().to(dtype)
    shape = (batch, seqlen, dim)
    y, bound = y.reshape(shape), bound.reshape(shape)
    if not channels_last:
        y, bound = y.transpose(1, 2), bound.transpose(1, 2)
    return y, bound, final


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, cu=None, slots=None, live=None,
         softplus=True, out=None, final=None):
    """Token-major scan. Returns (y, bound of y, final states, bound of the final states)."""
    dtype = u.dtype
    batch, seqlen, dim = u.shape
    N = A.shape[1]
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    G = B.shape[2]
    wide = lambda v: v.double().reshape(-1, G, N).repeat_interleave(dim // G, dim=1)  # noqa: E731
    Bw, Cw = wide(B), wide(C)
    uu = u.double().reshape(-1, dim)
    x = delta.double().reshape(-1, dim) + (0 if delta_bias is None else delta_bias.double())
    dt, dterr = x, U * x.abs()
    if softplus:
        dt = torch.logaddexp(x, torch.zeros_like(x))
        # slope at most 1 and at most dt itself below 0; the function's own error F
        dterr = torch.minimum(torch.ones_like(dt), dt) * U * (x.abs() + 1) + F * dt
    A = A.double()
    y = torch.zeros_like(uu) if out is None else out.double().reshape(-1, dim).clone()
    bound = torch.zeros_like(y)
    segs = sequences(batch, seqlen, cu)
    if final is None:
        final = torch.zeros((len(segs), dim, N)) if state is None or slots is None else state
    final = final.double().clone()
    ferr = torch.zeros_like(final)
    for i, (a, b) in enumerate(segs):
        row = row_of(i, slots, final.shape[0])
        h = torch.zeros((dim, N), dtype=torch.float64)
        if state is not None and row is not None and (live is None or int(live[i])):
            h = state[row].double().clone()
        mag, err = h.abs(), torch.zeros_like(h)  # magnitude of what is summed; error of h
        for t in range(a, b):
            d, e = dt[t].unsqueeze(1), dterr[t].unsqueeze(1)
            w = d * A
            decay = torch.exp(w)
            # the exponent is off by |A| err(dt) and two roundings of the product; exp by F on top
            rel = A.abs() * e + 2 * U * w.abs() * 2 + F
            inject = d * uu[t].unsqueeze(1) * Bw[t]
            ierr = (e * uu[t].unsqueeze(1) * Bw[t]).abs() + 3 * U * inject.abs()
            err = decay * (err + rel * mag) + ierr
            h = decay * h + inject
            mag = decay * mag + inject.abs()
            err = err + U * mag
            v = (Cw[t] * h).sum(1)
            verr = (Cw[t].abs() * err).sum(1) + (N + 2) * U * (Cw[t].abs() * mag).sum(1)
            if D is not None:
                v = v + D.double() * uu[t]
                verr = verr + 2 * U * (D.double() * uu[t]).abs()
            if z is not None:
                g, gerr = silu(z.double().reshape(-1, dim)[t], torch.zeros(dim, dtype=torch.float64))
                v, verr = v * g, verr * (g.abs() + gerr) + v.abs() * gerr + U * (v * g).abs()
            y[t], bound[t] = v, rounded(v, verr, dtype)
        if row is not None:
            final[row], ferr[row] = h, err + U * h.abs()
    return y.reshape(u.shape), bound.reshape(u.shape), final, ferr


def excess(got, want, bound):
    """Largest (|got - want| - bound) relative to the bound; negative or zero passes. Non-finite values have to agree."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    assert torch.equal(got[bad & ~torch.isnan(want)], want[bad & ~torch.isnan(want)]), "infinities differ"
    if bad.all():
        return 0.0
    d = (got - want).abs()[~bad]
    return float((d - bound[~bad]).max())
