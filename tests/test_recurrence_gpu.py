"""GatedRecurrenceFn, GatedRecurrenceGradFn and GatedRecurrenceUpdateFn on the GPU
against their float64 definitions (recurrence_reference.py, which also gives the
error bounds)."""

from __future__ import annotations

import pytest
import torch

import recurrence_reference as Q
import serving_reference as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def dev(t):
    return None if t is None else t.cuda()


def close(got, want, bound):
    e = R.excess(got, want, bound)
    assert e <= 0, f"off by {e} more than the bound"


def inputs(g, batch, seqlen, dim, dtype, bound=True):
    x, f = normal(g, batch, seqlen, dim, dtype=dtype), normal(g, batch, seqlen, dim, dtype=dtype, std=2.0, mean=2.0)
    return x, f, (torch.rand(dim, generator=g) * 0.95 if bound else None)


SHAPES = [(1, 1, 1), (2, 3, 5), (2, 130, 64), (3, 257, 48), (1, 700, 24), (2, 33, 130), (1, 16, 1027), (5, 1, 72),
          (1, 2100, 6), (70, 9, 66)]
PACKS = {
    "ragged": [0, 5, 5, 6, 140, 141, 143, 700],
    "empty ends": [0, 0, 0, 300, 300, 300],
    "ones": list(range(0, 41)),
    "single": [0, 513],
    "around blocks": [0, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 512, 513, 1023, 1024, 1025, 1500],
    "two long": [0, 1024, 2113],
    "nothing": [0, 0],
}


# ------------------------------------------------------------------ GatedRecurrenceFn


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,seqlen,dim", SHAPES)
@pytest.mark.parametrize("states", [False, True])
def test_batched(xm, cuda, dt, batch, seqlen, dim, states):
    g = gen(batch * 1000 + seqlen + dim)
    x, f, low = inputs(g, batch, seqlen, dim, DT[dt], bound=dim != 64)
    init = normal(g, batch, dim) if states else None
    y, bound, final, fb = Q.recurrence(x, f, low, init)
    if not states:
        close(xm.GatedRecurrenceFn(dev(x), dev(f), dev(low)), y, bound)
    got, state = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), output_final_state=1)
    close(got, y, bound)
    close(state, final, fb)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("pack", PACKS)
@pytest.mark.parametrize("dim", [40, 67, 130])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_packed_pool(xm, cuda, dt, pack, dim, index):
    """Packed sequences over a pool of slots, updated in place; rows behind the last sequence hold NaN and stay as they
    were; dead and unowned slots hold NaN too."""
    cu = PACKS[pack]
    units, behind = len(cu) - 1, 9
    g = gen(units * 31 + dim)
    x, f, low = inputs(g, 1, cu[-1] + behind, dim, DT[dt])
    x[:, cu[-1]:] = float("nan")
    f[:, cu[-1]:] = float("nan")
    slots = torch.randperm(units + 3, generator=g)[:units]
    live = torch.randint(0, 2, (units,), generator=g)
    pool = normal(g, units + 3, dim)
    pool[slots[live == 0]] = float("nan")
    if units > 2:
        slots[1], slots[2] = -1, units + 3
    before = torch.full_like(x, 7.0)
    y, bound, final, fb = Q.recurrence(x, f, low, pool, cu, slots, live, out=before)
    out, p = dev(before), dev(pool)
    got, state = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), p, torch.tensor(cu, dtype=index).cuda(),
                                      slots.to(index).cuda(), live.to(index).cuda(), output_final_state=1, out=out)
    assert got is out and state is p
    close(got, y, bound)
    close(p, final, fb)


@pytest.mark.parametrize("dim", [8, 200])
@pytest.mark.parametrize("inplace", [False, True])
def test_given_states(xm, cuda, dim, inplace):
    """Row states without slots, packed, in place or not: a long sequence in pieces."""
    g = gen(5)
    x, f, low = inputs(g, 1, 2600, dim, torch.float32)
    init = normal(g, 2, dim)
    y, bound, final, fb = Q.recurrence(x, f, low, init, [0, 1100, 2600])
    state = dev(init)
    for i, cuts in enumerate(((0, 300, 1100), (1100, 1108, 2600))):
        for a, b in zip(cuts, cuts[1:]):
            row = state[i:i + 1]
            kw = dict(final_state=row) if inplace else {}
            part, new = xm.GatedRecurrenceFn(dev(x[:, a:b]), dev(f[:, a:b]), dev(low), row, output_final_state=1, **kw)
            close(part, y[:, a:b], bound[:, a:b])
            if not inplace:
                state[i] = new[0]
    close(state, final, fb)
    both = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), torch.tensor([0, 1100, 2600]).cuda(),
                                output_final_state=1)
    close(both[0], y, bound)
    close(both[1], final, fb)


def test_long_memory(xm, cuda):
    """Gates near one carry the starting state across the whole length; f = 40 keeps it as it is."""
    g = gen(11)
    x, f, _ = inputs(g, 1, 5000, 6, torch.float32)
    f += 6
    f[:, :, 0] = 40
    init = normal(g, 1, 6) * 10
    y, bound, final, fb = Q.recurrence(x, f, None, init)
    got, state = xm.GatedRecurrenceFn(dev(x), dev(f), None, dev(init), output_final_state=1)
    close(got, y, bound)
    close(state, final, fb)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_extreme_gates(xm, cuda, dt):
    g = gen(12)
    x, f, low = inputs(g, 2, 300, 70, DT[dt])
    f[0, ::3] = 200
    f[0, 1::3] = -200
    f[1, ::5] = float("inf")
    f[1, 1::5] = -float("inf")
    low[:10] = 0.0
    low[10:20] = 0.99999
    init = normal(g, 2, 70)
    y, bound, final, fb = Q.recurrence(x, f, low, init)
    assert torch.isfinite(y).all()
    got, state = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), output_final_state=1)
    close(got, y, bound)
    close(state, final, fb)


def test_infinities_and_nan_stay_in_their_sequence(xm, cuda):
    """An infinite x or state lasts to its sequence's end, NaN too; neighbours in the row and other channels are as
    without them."""
    g = gen(13)
    cu = [0, 200, 201, 900, 1700, 2300]
    x, f, low = inputs(g, 1, 2300, 66, torch.float32)
    f.clamp_(-10, 10)  # gates below one in float32, and above zero
    init = normal(g, 5, 66)
    x[0, 100, 3] = float("inf")
    x[0, 200, 4] = float("nan")
    x[0, 1650, 65] = -float("inf")
    init[2, 5] = float("inf")
    init[4, 6] = float("nan")
    f[0, 905, 7] = float("nan")
    y, bound, final, fb = Q.recurrence(x, f, low, init, cu)
    got, state = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), torch.tensor(cu).cuda(), output_final_state=1)
    close(got, y, bound)
    close(state, final, fb)


def test_strided_and_misaligned_inputs(xm, cuda):
    g = gen(7)
    for dtype in DT.values():
        x, f, low = inputs(g, 2, 150, 64, dtype)
        init = dev(normal(g, 2, 64))
        want = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), init, output_final_state=1)
        wide = torch.cat([dev(x), dev(x)], 2)[..., :64]
        assert not wide.is_contiguous()
        got = xm.GatedRecurrenceFn(wide, dev(f).transpose(0, 1).contiguous().transpose(0, 1), dev(low), init,
                                   output_final_state=1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ref = Q.recurrence(x, f, low, init.cpu())
        for off in (1, 2, 3, 4):
            place = lambda t: torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape)  # noqa: E731
            xs, fs, ls, ss = (place(t) for t in (x, f, low, init))
            for d, s in ((xs, x), (fs, f), (ls, low), (ss, init)):
                d.copy_(s)
            o, last = place(x), place(init)
            got = xm.GatedRecurrenceFn(xs, fs, ls, ss, output_final_state=1, out=o, final_state=last)
            assert got[0] is o and got[1] is last
            close(o, *ref[:2])
            close(last, *ref[2:])


# ------------------------------------------------------------------ GatedRecurrenceGradFn


def _grad(xm, cu, dy, x, f, y, low, init, dlast, **kw):
    return xm.GatedRecurrenceGradFn(dev(dy), dev(x), dev(f), dev(y), dev(low), dev(init),
                                    None if cu is None else torch.tensor(cu).cuda(), dev(dlast), **kw)


def _grad_inputs(g, batch, seqlen, dim, dtype, cu=None, bound=True, states=True):
    x, f, low = inputs(g, batch, seqlen, dim, dtype, bound)
    units = batch if cu is None else len(cu) - 1
    init = normal(g, units, dim) if states else None
    y = Q.recurrence(x, f, low, init, cu)[0].to(dtype)
    return normal(g, batch, seqlen, dim, dtype=dtype), x, f, y, low, init, normal(g, units, dim) if states else None


def _close_grads(got, want, low, init):
    for k, (v, b) in enumerate(want):
        if (k == 2 and low is None) or (k == 3 and init is None):
            assert got[k] is None
        else:
            close(got[k], v, b)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,seqlen,dim", SHAPES)
@pytest.mark.parametrize("states", [False, True])
def test_grad_batched(xm, cuda, dt, batch, seqlen, dim, states):
    g = gen(batch * 100 + seqlen + dim)
    a = _grad_inputs(g, batch, seqlen, dim, DT[dt], bound=dim != 64, states=states)
    want = Q.recurrence_grad(*a[:6], None, a[6])
    _close_grads(_grad(xm, None, *a), want, a[4], a[5])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("pack", PACKS)
@pytest.mark.parametrize("dim", [40, 67, 130])
def test_grad_packed(xm, cuda, dt, pack, dim):
    """Rows behind the last sequence hold NaN and stay as they were."""
    cu = PACKS[pack]
    g = gen(len(cu) * 13 + dim)
    a = _grad_inputs(g, 1, cu[-1], dim, DT[dt], cu)
    pad = lambda t: torch.cat([t, torch.full((1, 9, dim), float("nan"), dtype=t.dtype)], 1)  # noqa: E731
    b = [pad(t) for t in a[:4]] + list(a[4:])
    want = Q.recurrence_grad(*a[:6], cu, a[6])
    before = torch.full_like(b[0], 7.0)
    outs = (dev(before), dev(before), None, None)
    got = _grad(xm, cu, *b, out=outs)
    assert got[0] is outs[0] and got[1] is outs[1]
    assert bool((got[0][:, cu[-1]:] == 7).all()) and bool((got[1][:, cu[-1]:] == 7).all())
    _close_grads([got[0][:, :cu[-1]], got[1][:, :cu[-1]], *got[2:]], want, a[4], a[5])
    # without the final states' gradients, and with a subset of the outputs
    want = Q.recurrence_grad(*a[:6], cu, None)
    got = xm.GatedRecurrenceGradFn(*[dev(t) for t in a[:6]], torch.tensor(cu, dtype=torch.int32).cuda(),
                                   output_lower_bound_grad=0)
    _close_grads(got, want, None, a[5])


def test_grad_requested_outputs(xm, cuda):
    """The starting states' gradient of sequences that start from zeros; none of the optional outputs."""
    g = gen(17)
    a = _grad_inputs(g, 2, 40, 24, torch.float32, states=False)
    want = Q.recurrence_grad(*a[:6], None, None)
    got = _grad(xm, None, *a, output_initial_state_grad=1)
    close(got[3], *want[3])
    got = _grad(xm, None, *a, output_lower_bound_grad=0)
    assert got[2] is None and got[3] is None
    close(got[0], *want[0])
    with pytest.raises(xm.XmError, match="requires a non-empty lower_bound"):
        _grad(xm, None, *a[:4], None, None, None, output_lower_bound_grad=1)


def test_grad_of_empty_sequences(xm, cuda):
    """No tokens: the states' gradient passes through, the lower bounds' is zero."""
    dl, low, init = torch.rand(3, 6, device="cuda"), torch.rand(6, device="cuda"), torch.rand(3, 6, device="cuda")
    e = torch.empty(3, 0, 6, device="cuda")
    dx, df, lb, d0 = xm.GatedRecurrenceGradFn(e, e, e, e, low, init, None, dl)
    assert dx.shape == e.shape and torch.equal(d0, dl) and torch.equal(lb, torch.zeros_like(low))
    e = torch.empty(0, 5, 6, device="cuda")
    dx, df, lb, d0 = xm.GatedRecurrenceGradFn(e, e, e, e, low, torch.empty(0, 6, device="cuda"))
    assert dx.shape == e.shape and d0.shape == (0, 6) and torch.equal(lb, torch.zeros_like(low))
    y, s = xm.GatedRecurrenceFn(e, e, low, output_final_state=1)
    assert y.shape == e.shape and s.shape == (0, 6)
    e = torch.empty(3, 0, 6, device="cuda")
    y, s = xm.GatedRecurrenceFn(e, e, low, init, output_final_state=1)
    assert torch.equal(s, init) and s is not init


def test_grad_extreme_gates_and_infinities(xm, cuda):
    g = gen(18)
    cu = [0, 200, 201, 900, 1300]
    dy, x, f, y, low, init, dl = _grad_inputs(g, 1, 1300, 66, torch.float32, cu)
    f.clamp_(-10, 10)
    f[0, ::7] = 200
    f[0, 1::7] = -200
    y = Q.recurrence(x, f, low, init, cu)[0].to(torch.float32)
    f2 = f.clone()
    want = Q.recurrence_grad(dy, x, f2, y, low, init, cu, dl)
    _close_grads(_grad(xm, cu, dy, x, f2, y, low, init, dl), want, low, init)
    dy[0, 850, 3] = float("inf")
    dl[0, 4] = float("nan")
    dy[0, 1000, 64] = float("nan")
    f2 = f.clamp(-10, 10)  # where a or 1 - a is zero, infinity times it is NaN or not by one rounding
    want = Q.recurrence_grad(dy, x, f2, y, low, init, cu, dl)
    _close_grads(_grad(xm, cu, dy, x, f2, y, low, init, dl), want, low, init)


@pytest.mark.parametrize("batch,seqlen,dim", [(1, 700, 70), (2, 100, 40), (160, 270, 9)])
def test_lower_bounds_of_one(xm, cuda, batch, seqlen, dim):
    """Such a channel keeps its state for good; its bound has a gradient, its inputs have (next to) none."""
    g = gen(20)
    x, f, low = inputs(g, batch, seqlen, dim, torch.float32)
    ones = torch.arange(dim) % 3 == 1
    low[ones] = 1.0
    init, dl = normal(g, batch, dim), normal(g, batch, dim)
    y, last = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), output_final_state=1)
    want = Q.recurrence(x, f, low, init)
    close(y, *want[:2])
    assert torch.equal(y[..., ones].cpu(), init[:, None, ones].expand(-1, seqlen, -1))
    dy = normal(g, batch, seqlen, dim)
    want = Q.recurrence_grad(dy, x, f, y.cpu(), low, init, None, dl)
    # G is at most the sum of |dy| and |dl|, h - x at most 12: times 2^-60
    most = 12 * (dy.abs().sum(1).max() + dl.abs().max()).double() * 2.0**-60
    for v, b in want[:2]:
        b[..., ones] += most
    got = _grad(xm, None, dy, x, f, y.cpu(), low, init, dl)
    _close_grads(got, want, low, init)


def test_grad_misaligned(xm, cuda):
    g = gen(19)
    for dtype in DT.values():
        a = _grad_inputs(g, 2, 140, 64, dtype)
        want = Q.recurrence_grad(*a[:6], None, a[6])
        for off in (1, 2, 4):
            place = lambda t: torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape)  # noqa: E731
            moved = [place(t) for t in a]
            for d, s in zip(moved, a):
                d.copy_(s)
            outs = (place(a[0]), place(a[0]), place(a[4]), place(a[5]))
            got = xm.GatedRecurrenceGradFn(*moved[:6], None, moved[6], out=outs)
            assert all(p is q for p, q in zip(got, outs))
            _close_grads(got, want, a[4], a[5])


# ------------------------------------------------------------------ GatedRecurrenceUpdateFn


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,dim", [(1, 1), (3, 67), (5, 72), (2, 1024), (17, 4096), (300, 66), (1, 4099)])
@pytest.mark.parametrize("pool", [False, True])
def test_update(xm, cuda, dt, batch, dim, pool):
    g = gen(batch + dim)
    x, f, low = inputs(g, batch, 1, dim, DT[dt], bound=dim != 72)
    n = batch + 4 if pool else batch
    state = normal(g, n, dim)
    slots = torch.randperm(n, generator=g)[:batch] if pool else None
    if pool and batch > 2:
        slots[0], slots[1] = -1, n
    before = torch.full((batch, 1, dim), 3.0, dtype=DT[dt])
    y, bound, final, fb = Q.recurrence(x, f, low, state, None, slots, final=state)
    if pool and batch > 2:
        y[:2], bound[:2] = 3.0, 0.0
    out, s = dev(before[:, 0]), dev(state)
    got, new = xm.GatedRecurrenceUpdateFn(dev(x[:, 0]), dev(f[:, 0]), dev(low), s, dev(slots), out=out)
    assert got is out and new is s
    close(got, y[:, 0], bound[:, 0])
    close(s, final, fb)
    if not pool:
        kept, other = dev(state), torch.empty_like(s)
        got2, new2 = xm.GatedRecurrenceUpdateFn(dev(x[:, 0]), dev(f[:, 0]), dev(low), kept, new_state=other)
        assert new2 is other and torch.equal(other, s) and torch.equal(kept.cpu(), state) and torch.equal(got2, got)


def test_update_misaligned(xm, cuda):
    g = gen(23)
    for dtype in DT.values():
        x, f, low = inputs(g, 5, 1, 64, dtype)
        state = normal(g, 9, 64)
        slots = torch.tensor([8, 0, 3, -5, 4])
        y, bound, final, fb = Q.recurrence(x, f, low, state, None, slots, final=state)
        y[3], bound[3] = 2.0, 0.0  # no slot: the row stays as it was
        for off in (1, 2, 3):
            place = lambda t: torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape)  # noqa: E731
            moved = [place(t) for t in (x[:, 0], f[:, 0], low, state, x[:, 0])]
            for d, s in zip(moved, (x[:, 0], f[:, 0], low, state, torch.full_like(x[:, 0], 2.0))):
                d.copy_(s)
            xm.GatedRecurrenceUpdateFn(*moved[:4], slots.cuda(), out=moved[4])
            close(moved[4], y[:, 0], bound[:, 0])
            close(moved[3], final, fb)


def test_a_row_does_not_depend_on_its_batch(xm, cuda):
    g = gen(24)
    x, f, low = inputs(g, 600, 1, 192, torch.bfloat16)
    x, f, low, state = dev(x[:, 0]), dev(f[:, 0]), dev(low), dev(normal(g, 600, 192))
    y, new = xm.GatedRecurrenceUpdateFn(x, f, low, state.clone())
    for rows in (slice(0, 1), slice(7, 40), slice(599, 600)):
        y1, n1 = xm.GatedRecurrenceUpdateFn(x[rows], f[rows], low, state[rows].clone())
        assert torch.equal(y1, y[rows]) and torch.equal(n1, new[rows])


# ------------------------------------------------------------------ together, streams, graphs


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_prompt_then_tokens(xm, cuda, dt):
    """Packed prompts into a pool, then tokens one by one: each sequence's outputs are the whole sequence's."""
    g = gen(31)
    lens, extra, dim = [5, 40, 1, 130], 6, 72
    whole = [inputs(g, 1, n + extra, dim, DT[dt])[:2] for n in lens]
    low = torch.rand(dim, generator=g) * 0.9
    pool = torch.full((6, dim), float("nan"), device="cuda")
    slots = torch.tensor([4, 1, 0, 5], dtype=torch.int32).cuda()
    live = torch.zeros(4, dtype=torch.int32).cuda()
    cu = torch.tensor([0, 5, 45, 46, 176], dtype=torch.int32).cuda()
    head = [torch.cat([w[k][:, :n] for w, n in zip(whole, lens)], 1).cuda() for k in (0, 1)]
    y, _ = xm.GatedRecurrenceFn(*head, dev(low), pool, cu, slots, live, output_final_state=1)
    steps = []
    for t in range(extra):
        tok = [torch.cat([w[k][:, n + t] for w, n in zip(whole, lens)]).cuda() for k in (0, 1)]
        steps.append(xm.GatedRecurrenceUpdateFn(*tok, dev(low), pool, slots)[0])
    for i, n in enumerate(lens):
        want, bound, final, fb = Q.recurrence(*whole[i], low)
        a = int(cu[i])
        close(y[:, a:a + n], want[:, :n], bound[:, :n])
        close(torch.stack([s[i] for s in steps]).unsqueeze(0), want[:, n:], bound[:, n:])
        close(pool[int(slots[i])], final[0], fb[0])


def _mm(a, b):
    """a @ b without a library product, which may sum through a workspace that captured graphs share."""
    return (a.unsqueeze(-1) * b).sum(-2)


def _outer(a, b):
    return (a.unsqueeze(-1) * b.unsqueeze(-2)).sum((0, 1))


def _training_step(xm, p):
    """Norm with the residual, two projections, recurrence; and back."""
    h, s, stats = xm.LayerNormFn(p["x"], p["w"], p["b"], p["r"], output_stats=1)
    xin, f = _mm(h, p["wx"]), _mm(h, p["wf"])
    y, last = xm.GatedRecurrenceFn(xin, f, p["low"], p["h0"], p["cu"], output_final_state=1)
    dx, df, dlow, dh0 = xm.GatedRecurrenceGradFn(p["dy"], xin, f, y, p["low"], p["h0"], p["cu"], p["dl"])
    dh = _mm(dx, p["wx"].t()) + _mm(df, p["wf"].t())
    ds, dw, db = xm.LayerNormGradFn(dh, s, p["w"], stats, p["ds"], output_bias_grad=1)
    return dict(y=y, s=s, last=last, dlow=dlow, dh0=dh0, ds=ds, dw=dw, db=db,
                dwx=_outer(h, dx), dwf=_outer(h, df))


def _training_inputs(seed, dim=96, cu=(0, 300, 301, 777)):
    g = gen(seed)
    n = cu[-1]
    p = dict(x=normal(g, 1, n, dim), r=normal(g, 1, n, dim), w=normal(g, dim, std=0.1, mean=1.0), b=normal(g, dim, std=0.1),
             wx=normal(g, dim, dim, std=dim**-0.5), wf=normal(g, dim, dim, std=dim**-0.5), low=torch.rand(dim, generator=g),
             h0=normal(g, len(cu) - 1, dim), dy=normal(g, 1, n, dim), dl=normal(g, len(cu) - 1, dim), ds=normal(g, 1, n, dim))
    p["low"] *= 0.9
    p = {k: v.cuda() for k, v in p.items()}
    p["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
    return p


def test_training_step_against_autograd(xm, cuda):
    """A layer forward and backward in float32 against autograd over the formulas in float64. Every operator is off by
    about 2^-20 of what it sums; gates of at most 1 - 0.1 / (1 + e^5) keep at most some hundred tokens, whose errors
    add up to 2^-13 of the largest value at the very most."""
    p = _training_inputs(41)
    got = _training_step(xm, p)
    leaves = {k: p[k].double().requires_grad_() for k in ("x", "r", "w", "b", "wx", "wf", "low", "h0")}
    s = leaves["x"] + leaves["r"]
    mean = s.mean(-1, keepdim=True)
    h = (s - mean) * torch.rsqrt(((s - mean) ** 2).mean(-1, keepdim=True) + 1e-5) * leaves["w"] + leaves["b"]
    xin, a = h @ leaves["wx"], leaves["low"] + (1 - leaves["low"]) * torch.sigmoid(h @ leaves["wf"])
    ys, last = [], []
    cu = p["cu"].tolist()
    for i, (b, e) in enumerate(zip(cu, cu[1:])):
        state = leaves["h0"][i]
        for t in range(b, e):
            state = a[0, t] * state + (1 - a[0, t]) * xin[0, t]
            ys.append(state)
        last.append(state)
    y, last = torch.stack(ys).unsqueeze(0), torch.stack(last)
    loss = (y * p["dy"]).sum() + (last * p["dl"]).sum() + (s * p["ds"]).sum()
    want = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    pairs = dict(y=y, last=last, s=s, ds=want["x"], dw=want["w"], db=want["b"], dwx=want["wx"], dwf=want["wf"],
                 dlow=want["low"], dh0=want["h0"])
    assert torch.equal(want["x"], want["r"])
    for k, v in pairs.items():
        v = v.detach()
        assert float((got[k].double() - v).abs().max()) <= 2.0**-13 * float(v.abs().max()), k


def _differing(a, b):
    return [k for k in a if not torch.equal(a[k], b[k])]


def test_streams_and_two_calls_at_once(xm, cuda):
    p, q = _training_inputs(42), _training_inputs(43, dim=160, cu=(0, 2000))
    wp, wq = _training_step(xm, p), _training_step(xm, q)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = _training_step(xm, p)
        with torch.cuda.stream(s2):
            b = _training_step(xm, q)
        torch.cuda.synchronize()
        assert not _differing(a, wp) and not _differing(b, wq)
    # a stream by argument
    want = xm.GatedRecurrenceFn(p["x"], p["r"], p["low"], p["h0"], p["cu"])
    got = xm.GatedRecurrenceFn(p["x"], p["r"], p["low"], p["h0"], p["cu"], stream=s1)
    g2 = xm.GatedRecurrenceGradFn(p["dy"], p["x"], p["r"], want, p["low"], p["h0"], p["cu"], stream=s2)
    g1 = xm.GatedRecurrenceGradFn(p["dy"], p["x"], p["r"], want, p["low"], p["h0"], p["cu"])
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(u, v) for u, v in zip(g1, g2))


def test_captured_graphs(xm, cuda):
    """Two captured training steps replayed in turn and on two streams at once, with inputs that change in place."""
    p, q = _training_inputs(44), _training_inputs(45, dim=160, cu=(0, 1500))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for v in (p, q):
            _training_step(xm, v)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = _training_step(xm, v)
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for step in range(4):
        for v in (p, q):
            v["x"].mul_(-0.9)
            v["dy"].add_(0.1)
        torch.cuda.synchronize()
        if step % 2:
            with torch.cuda.stream(side):
                graphs[0][0].replay()
            graphs[1][0].replay()
        else:
            graphs[1][0].replay()
            graphs[0][0].replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for (_, out), v in zip(graphs, (p, q)):
                assert not _differing(out, _training_step(xm, v))


def test_repeatable_bits(xm, cuda):
    p = _training_inputs(46, dim=200, cu=(0, 40, 1700))
    want = _training_step(xm, p)
    for _ in range(20):
        assert not _differing(_training_step(xm, p), want)


# ------------------------------------------------------------------ many and few rows, short and long

# (batch, seqlen, dim) or (offsets, None, dim); a row's 64 channels are a warp's or a block's
CUTS = {
    "blocks of eight, words": (3, 300, 3264),
    "blocks of eight, odd rows": (3, 300, 3267),
    "blocks of eight, pairs": (3, 300, 3266),
    "blocks of four, words": (5, 260, 4000),
    "blocks of four, pairs": (5, 261, 3998),
    "blocks of four, odd rows": (5, 261, 3999),
    "packed, blocks of eight": ([0, 0, 7, 8, 9, 128, 128, 256, 257, 530, 600], None, 9600),
    "packed, blocks of eight, odd rows": ([3, 4, 100, 411], None, 9607),
    "packed, blocks of four": ([0, 1, 130, 131, 330, 400], None, 19001),
    "a block for each SM": (2, 500, 3904),
    "a warp for each row": (3, 200, 3265),
    "a warp for each row, pairs": (3, 200, 3266),
    "short rows of two sequences": (9, 32, 70),
    "short rows, in turns": (290, 32, 64),
    "segments of several rows": (2, 1200, 130),
    "segments, words": (2, 1200, 136),
}


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cut", CUTS)
def test_every_cut(xm, cuda, dt, cut):
    """Forward and backward, at sizes that are cut in every way there is; repeated, and from a captured graph."""
    batch, seqlen, dim = CUTS[cut]
    cu = batch if seqlen is None else None
    if cu is not None:
        batch, seqlen = 1, cu[-1] + 5
    g = gen(dim + seqlen)
    x, f, low = inputs(g, batch, seqlen, dim, DT[dt])
    units = batch if cu is None else len(cu) - 1
    init, dl = normal(g, units, dim), normal(g, units, dim)
    hole = torch.full_like(x, 7.0)
    y, bound, final, fb = Q.recurrence(x, f, low, init, cu, out=hole)
    ys = y.to(DT[dt])
    dy = normal(g, batch, seqlen, dim, dtype=DT[dt])
    want = Q.recurrence_grad(dy, x, f, ys, low, init, cu, dl, dx=hole, df=hole)
    c = None if cu is None else torch.tensor(cu).cuda()
    a = [dev(t) for t in (x, f, low, init, ys, dy, dl)]
    outs = [torch.full_like(a[0], 7.0) for _ in range(3)]

    def run():
        got = xm.GatedRecurrenceFn(a[0], a[1], a[2], a[3], c, output_final_state=1, out=outs[0])
        return (*got, *xm.GatedRecurrenceGradFn(a[5], a[0], a[1], a[4], a[2], a[3], c, a[6],
                                                out=(outs[1], outs[2], None, None)))

    got = run()
    close(got[0], y, bound)
    close(got[1], final, fb)
    _close_grads(got[2:], want, low, init)
    first = [t.clone() for t in got]
    assert all(torch.equal(u, v) for u, v in zip(run(), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = run()
    for t in outs:
        t.fill_(7.0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(again, first))


@pytest.mark.parametrize("dim", [9600, 19001])
def test_infinities_in_rows_of_blocks(xm, cuda, dim):
    """What is infinite or NaN lasts to its sequence's end and touches no other sequence or channel."""
    g = gen(dim)
    cu = [0, 140, 141, 400]
    dy, x, f, _, low, init, dl = _grad_inputs(g, 1, 400, dim, torch.float32, cu)
    f.clamp_(-10, 10)
    x[0, 20, 3], x[0, 140, 4], x[0, 200, dim - 1] = float("inf"), float("nan"), -float("inf")
    init[2, 5], init[0, 6] = float("inf"), float("nan")
    y, bound, final, fb = Q.recurrence(x, f, low, init, cu)
    c = torch.tensor(cu).cuda()
    got, last = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), c, output_final_state=1)
    close(got, y, bound)
    close(last, final, fb)
    dy, x, f, y, low, init, dl = _grad_inputs(g, 1, 400, dim, torch.float32, cu)
    f.clamp_(-10, 10)
    y = Q.recurrence(x, f, low, init, cu)[0].float()
    dy[0, 350, 3], dy[0, 100, dim - 1], dl[2, 64], dl[0, 70] = float("inf"), float("nan"), -float("inf"), float("nan")
    want = Q.recurrence_grad(dy, x, f, y, low, init, cu, dl)
    _close_grads(_grad(xm, cu, dy, x, f, y, low, init, dl), want, low, init)


@pytest.mark.parametrize("seqlen,dim", [(256, 6), (130, 70)])
def test_more_rows_than_partial_sums(xm, cuda, seqlen, dim):
    """A row's results do not depend on how many rows there are, and the lower bounds' gradient is the sum over them."""
    g = gen(61)
    n, part = 2300, 460
    x, f, low = (dev(t) for t in inputs(g, n, seqlen, dim, torch.bfloat16))
    dy, init, dl = (dev(normal(g, *s, dtype=t)) for s, t in (((n, seqlen, dim), torch.bfloat16),
                                                             ((n, dim), torch.float32), ((n, dim), torch.float32)))
    y, last = xm.GatedRecurrenceFn(x, f, low, init, output_final_state=1)
    got = xm.GatedRecurrenceGradFn(dy, x, f, y, low, init, None, dl)
    total = torch.zeros(dim, dtype=torch.float64)
    for i in range(0, n, part):
        r = slice(i, i + part)
        yr, lr = xm.GatedRecurrenceFn(x[r], f[r], low, init[r], output_final_state=1)
        assert torch.equal(yr, y[r]) and torch.equal(lr, last[r])
        gr = xm.GatedRecurrenceGradFn(dy[r], x[r], f[r], y[r], low, init[r], None, dl[r])
        assert torch.equal(gr[0], got[0][r]) and torch.equal(gr[1], got[1][r]) and torch.equal(gr[3], got[3][r])
        total += gr[2].cpu().double()
    # the terms, G (h - x) sigmoid(-f) = df / ((1 - low) sigmoid(f)) with df rounded to bfloat16, are the same bits in both;
    # a warp adds those of at most three rows in a row, and a column's sum fewer than 100 of such: below 1024 roundings
    mag = (got[1].double().abs() / ((1 - low.double()) * torch.sigmoid(f.double()))).sum((0, 1)).cpu() * 1.01
    close(got[2], total, 2 * 1024 * 2.0**-24 * mag)


# ------------------------------------------------------------------ sizes and indices at the edges


def test_offsets_past_32_bits(xm, cuda):
    """Tensors of more than 2^31 elements: a sequence whose tokens lie behind that, and a pool's last slots."""
    dim, tokens = 4096, 2**19 + 300
    x = torch.zeros(1, tokens, dim, dtype=torch.bfloat16, device="cuda")
    f = torch.zeros(1, tokens, dim, dtype=torch.bfloat16, device="cuda")
    g = gen(51)
    a = 2**19 - 100
    xs, fs, low = inputs(g, 1, 390, dim, torch.bfloat16)
    x[:, a:a + 390], f[:, a:a + 390] = xs.cuda(), fs.cuda()
    cu = torch.tensor([a, a + 390]).cuda()
    init = normal(g, 1, dim)
    y, bound, final, fb = Q.recurrence(xs, fs, low, init)
    out, last = xm.GatedRecurrenceFn(x, f, dev(low), dev(init), cu, output_final_state=1, out=torch.zeros_like(x))
    close(out[:, a:a + 390], y, bound)
    close(last, final, fb)
    assert not bool(out[:, :a].any()) and not bool(out[:, a + 390:].any())
    dys, dl = normal(g, 1, 390, dim, dtype=torch.bfloat16), normal(g, 1, dim)
    ys = y.to(torch.bfloat16)
    want = Q.recurrence_grad(dys, xs, fs, ys, low, init, None, dl)
    dy, yy = torch.zeros_like(x), out
    dy[:, a:a + 390], yy[:, a:a + 390] = dys.cuda(), ys.cuda()
    got = xm.GatedRecurrenceGradFn(dy, x, f, yy, dev(low), dev(init), cu, dev(dl))
    _close_grads([got[0][:, a:a + 390], got[1][:, a:a + 390], *got[2:]], want, low, init)
    del x, f, out, dy, yy, got
    slots = 2**19 + 7
    pool = torch.zeros(slots, dim, device="cuda")
    idx = torch.tensor([slots - 1, 3, 2**19 + 1])
    rows = normal(g, 3, dim)
    pool[idx.cuda()] = rows.cuda()
    xs, fs, low = inputs(g, 3, 1, dim, torch.float32)
    y, bound, final, fb = Q.recurrence(xs, fs, low, rows)
    got, _ = xm.GatedRecurrenceUpdateFn(dev(xs[:, 0]), dev(fs[:, 0]), dev(low), pool, idx.cuda())
    close(got, y[:, 0], bound[:, 0])
    close(pool[idx.cuda()], final, fb)


def test_more_sequences_than_a_grid_dimension(xm, cuda):
    n, dim = 70000, 3
    g = gen(52)
    x, f, low = inputs(g, n, 2, dim, torch.float32)
    init = normal(g, n, dim)
    a = low + (1 - low) * torch.sigmoid(f.double())
    u = (1 - low) * torch.sigmoid(-f.double())
    h1 = a[:, 0] * init + u[:, 0] * x[:, 0]
    want = torch.stack([h1, a[:, 1] * h1 + u[:, 1] * x[:, 1]], 1)
    # two steps of values below 10: some 30 roundings of at most 2^-21 each
    bound = torch.full_like(want, 10 * 30 * 2.0**-21)
    got, last = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), output_final_state=1)
    close(got, want, bound)
    close(last, want[:, 1], bound[:, 1])
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32).cuda()
    flat = lambda t: dev(t).view(1, 2 * n, dim)  # noqa: E731
    got, last = xm.GatedRecurrenceFn(flat(x), flat(f), dev(low), dev(init), cu, output_final_state=1)
    close(got.view(n, 2, dim), want, bound)
    close(last, want[:, 1], bound[:, 1])
    dy = normal(g, n, 2, dim)
    for packed in (False, True):
        y = want.float()
        args = [flat(t) if packed else dev(t) for t in (dy, x, f, y)]
        got = xm.GatedRecurrenceGradFn(*args, dev(low), dev(init), cu if packed else None)
        G1 = dy[:, 1].double()
        G0 = dy[:, 0] + a[:, 1] * G1
        G = torch.stack([G0, G1], 1)
        d = torch.stack([init, y[:, 0]], 1).double() - x
        s = torch.sigmoid(f.double())
        close(got[0].view(n, 2, dim), u * G, bound)
        close(got[1].view(n, 2, dim), G * d * u * s, 10 * bound)
        terms = G * d * torch.sigmoid(-f.double())
        close(got[2], terms.sum((0, 1)), terms.abs().sum((0, 1)) * 2 * n * 2.0**-24)
        close(got[3], a[:, 0] * G0, bound[:, 0])
    tok = xm.GatedRecurrenceUpdateFn(dev(x[:, 0]), dev(f[:, 0]), dev(low), dev(init))
    close(tok[0], h1, bound[:, 0])


def test_a_slot_named_twice_touches_nothing_else(xm, cuda):
    g = gen(53)
    x, f, low = inputs(g, 1, 60, 40, torch.float32)
    pool = normal(g, 6, 40).cuda()
    kept = pool.clone()
    slots = torch.tensor([2, 2, 4]).cuda()
    xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), pool, torch.tensor([0, 20, 40, 60]).cuda(), slots, output_final_state=1)
    others = [0, 1, 3, 5]
    assert torch.equal(pool[others], kept[others])
    xm.GatedRecurrenceUpdateFn(dev(x[0, :3]), dev(f[0, :3]), dev(low), pool, slots)
    assert torch.equal(pool[others], kept[others])


def test_refusals_on_the_device(xm, cuda):
    from types import SimpleNamespace

    x, s = torch.rand(2, 20, 8, device="cuda"), torch.rand(2, 8, device="cuda")
    fn, grad, tok = xm.GatedRecurrenceFn, xm.GatedRecurrenceGradFn, xm.GatedRecurrenceUpdateFn
    wide = torch.rand(2, 16, device="cuda")[:, :8]
    other = SimpleNamespace(device_index=1, cuda_stream=torch.cuda.default_stream(0).cuda_stream)
    for call, match in (
        (lambda: fn(x, x.cpu()), "f must be a tensor on cuda:0"),
        (lambda: fn(x, None), "f shape must match x"),
        (lambda: fn(x, x.half()), "float32"),
        (lambda: fn(x, x, None, s.half()), "initial_state must be float32"),
        (lambda: fn(x, x, out=x), "an output must not overlap an input"),
        (lambda: fn(x, x, out=torch.empty(2, 20, 16, device="cuda")[..., :8]), "out must be a contiguous tensor"),
        (lambda: fn(x, x, None, wide, final_state=wide, output_final_state=1), "updated in place and must be contiguous"),
        (lambda: fn(x, x, stream=other), "stream belongs to another device"),
        (lambda: grad(x, x, x, x, stream=other), "stream belongs to another device"),
        (lambda: grad(x, x, x, x, out=(x, None, None, None)), "an output must not overlap an input"),
        (lambda: grad(x, x, x, x.half()), "float32"),
        (lambda: grad(x, x, x, x, out=(x.half(), None, None, None)), "output must have the shape and type of dy"),
        (lambda: tok(x[:, 0], x[:, 0], None, wide), "updated in place and must be contiguous"),
        (lambda: tok(x[:, 0].contiguous(), x[:, 0], None, s[:1]), "state must have shape"),
    ):
        with pytest.raises(xm.XmError, match=match):
            call()


def test_malformed_offsets_stay_inside(xm, cuda):
    """Offsets that descend or point outside give undefined values, but only inside the outputs."""
    g = gen(54)
    x, f, low = (t.cuda() for t in inputs(g, 1, 500, 40, torch.float32))
    guard = torch.full((3, 500, 40), 5.0, device="cuda")
    pool = torch.full((9, 40), 5.0, device="cuda")
    for cu in ([0, 900, 300, 500], [-7, 100, 2000, 499], [400, 100, 50, 10], [500, 500, 500, 500], [10, 20, 15, 490]):
        c = torch.tensor(cu).cuda()
        xm.GatedRecurrenceFn(x, f, low, pool[3:6], c, output_final_state=1, out=guard[1:2], final_state=pool[3:6])
        xm.GatedRecurrenceGradFn(x, x, f, x, low, pool[3:6].clone(), c, out=(guard[1:2], None, None, None))
        torch.cuda.synchronize()
        assert bool((guard[::2] == 5).all()) and bool((pool[:3] == 5).all()) and bool((pool[6:] == 5).all())


@pytest.mark.parametrize("dt,tokens,dim", [("bf16", 300, 72), ("bf16", 300, 71), ("f32", 40, 33), ("bf16", 300, 9600),
                                           ("f32", 300, 9607), ("bf16", 280, 19001)])
def test_malformed_offsets_in_every_cut(xm, cuda, dt, tokens, dim):
    """The same where a block, or its warps in turn, takes a row: every call ends and stays inside its outputs."""
    g = gen(55)
    x, f, low = (t.cuda() for t in inputs(g, 1, tokens, dim, DT[dt]))
    guard = torch.full((3, tokens, dim), 5.0, dtype=DT[dt], device="cuda")
    pool = torch.full((9, dim), 5.0, device="cuda")
    for cu in ([0, 900, 30, tokens], [-7, 100, 2000, tokens - 1], [tokens - 10, 30, 20, 10], [tokens] * 4, [10, 20, 15, 36],
               [5, 4, 3, tokens]):
        c = torch.tensor(cu).cuda()
        xm.GatedRecurrenceFn(x, f, low, pool[3:6], c, output_final_state=1, out=guard[1:2], final_state=pool[3:6])
        xm.GatedRecurrenceGradFn(x, x, f, x, low, pool[3:6].clone(), c, out=(guard[1:2], None, None, None))
        torch.cuda.synchronize()
        assert bool((guard[::2] == 5).all()) and bool((pool[:3] == 5).all()) and bool((pool[6:] == 5).all())
    # and the next call is as it should be
    y, bound, final, fb = Q.recurrence(x.cpu(), f.cpu(), low.cpu())
    got, last = xm.GatedRecurrenceFn(x, f, low, output_final_state=1)
    close(got, y, bound)
    close(last, final, fb)


@pytest.mark.parametrize("dim", [61, 66, 71])
def test_views_at_the_ends_of_a_buffer(xm, cuda, dim):
    """Tensors that begin off a 16-byte word and end with the buffer's last element, between neighbours that hold NaN."""
    g = gen(56)
    for dtype in DT.values():
        for n, off in ((1, 1), (40, 3), (130, 7)):
            x, f, low = inputs(g, 1, n, dim, dtype)
            init, dl = normal(g, 1, dim), normal(g, 1, dim)
            y, bound, final, fb = Q.recurrence(x, f, low, init)
            dy, ys = normal(g, 1, n, dim, dtype=dtype), y.to(dtype)
            want = Q.recurrence_grad(dy, x, f, ys, low, init, None, dl)

            def place(t):
                buf = torch.full((off + t.numel(),), float("nan"), dtype=t.dtype, device="cuda")
                buf[off:] = t.flatten().cuda()
                return buf[off:].view(t.shape)

            a = [place(t) for t in (x, f, low, init, ys, dy, dl)]
            got, last = xm.GatedRecurrenceFn(*a[:4], output_final_state=1)
            close(got, y, bound)
            close(last, final, fb)
            _close_grads(xm.GatedRecurrenceGradFn(a[5], a[0], a[1], a[4], a[2], a[3], None, a[6]), want, low, init)


def test_long_rows_of_few_channels(xm, cuda):
    """Rows that are cut into as many segments as there may be."""
    for dt, n, dim, cu in ((torch.float32, 7000, 7, [0, 1, 3500, 7000]), (torch.bfloat16, 9001, 64, [0, 9001])):
        a = _grad_inputs(gen(57), 1, n, dim, dt, cu)
        dy, x, f, ys, low, init, dl = a
        y, bound, final, fb = Q.recurrence(x, f, low, init, cu)
        got, last = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), dev(init), torch.tensor(cu).cuda(), output_final_state=1)
        close(got, y, bound)
        close(last, final, fb)
        _close_grads(_grad(xm, cu, *a), Q.recurrence_grad(*a[:6], cu, dl), low, init)
