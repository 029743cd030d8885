"""CausalConv1dFn, CausalConv1dUpdateFn, SelectiveScanVarlenFn and
SelectiveStateUpdateFn on the GPU against their float64 definitions
(serving_reference.py, which also gives the error bounds)."""

from __future__ import annotations

import pytest
import torch

import serving_reference as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def dev(t):
    return None if t is None else t.cuda()


def close(got, want, bound):
    e = R.excess(got, want, bound)
    assert e <= 0, f"off by {e} more than the bound"


def conv_inputs(g, batch, seqlen, dim, width, dtype, channels_last, bias=True):
    x = normal(g, *((batch, seqlen, dim) if channels_last else (batch, dim, seqlen)), dtype=dtype)
    w = (torch.rand(dim, width, generator=g) - 0.5) * 2 * width**-0.5
    return x, w, (torch.rand(dim, generator=g) - 0.5 if bias else None)


def scan_inputs(g, batch, seqlen, dim, N, dtype, groups=1, gate=True, skip=True, bias=True, softplus=True):
    x = dict(u=normal(g, batch, seqlen, dim, dtype=dtype), delta=normal(g, batch, seqlen, dim, dtype=dtype))
    if not softplus:
        x["delta"] = (torch.rand(batch, seqlen, dim, generator=g) * 0.2).to(dtype)
    x["A"] = -(torch.rand(dim, N, generator=g) * N + 0.05)
    x["B"], x["C"] = normal(g, batch, seqlen, groups, N, dtype=dtype), normal(g, batch, seqlen, groups, N, dtype=dtype)
    x["D"] = normal(g, dim) if skip else None
    x["z"] = normal(g, batch, seqlen, dim, dtype=dtype) if gate else None
    x["delta_bias"] = (normal(g, dim) - 2 if softplus else torch.rand(dim, generator=g) * 0.1) if bias else None
    return x


SCAN = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


# ------------------------------------------------------------------ CausalConv1dFn


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("channels_last", [0, 1])
@pytest.mark.parametrize("batch,seqlen,dim,width", [(1, 1, 1, 4), (2, 3, 5, 4), (3, 257, 64, 4), (2, 1000, 72, 3),
                                                    (1, 2048, 8, 2), (2, 65, 1027, 4), (1, 16, 4096, 4)])
def test_conv_batched(xm, cuda, dt, channels_last, batch, seqlen, dim, width):
    g = gen(batch * 1000 + seqlen + dim)
    x, w, b = conv_inputs(g, batch, seqlen, dim, width, DT[dt], channels_last, bias=dim != 64)
    y, bound, final = R.conv(x, w, b, channels_last=channels_last, silu_=seqlen != 1000)
    got, state = xm.CausalConv1dFn(dev(x), dev(w), dev(b), silu=int(seqlen != 1000), channels_last=channels_last,
                                   output_final_state=1)
    close(got, y, bound)
    assert torch.equal(state.cpu(), final)
    assert torch.equal(xm.CausalConv1dFn(dev(x), dev(w), dev(b), silu=int(seqlen != 1000),
                                         channels_last=channels_last), got)


PACKS = {
    "ragged": [0, 5, 5, 6, 140, 141, 143, 700],
    "empty ends": [0, 0, 0, 300, 300, 300],
    "ones": list(range(0, 41)),
    "single": [0, 513],
    "around tiles": [0, 31, 64, 97, 127, 128, 129, 255, 256, 258, 513],
    "nothing": [0, 0],
}


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("channels_last", [0, 1])
@pytest.mark.parametrize("pack", PACKS)
@pytest.mark.parametrize("dim", [40, 67])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_conv_packed_pool(xm, cuda, dt, channels_last, pack, dim, index):
    """Packed sequences over a pool of slots, updated in place; rows behind the last sequence hold NaN and stay as they
    were; dead and unowned slots hold NaN too."""
    cu = PACKS[pack]
    units, behind = len(cu) - 1, 9
    g = gen(units * 31 + dim)
    x, w, b = conv_inputs(g, 1, cu[-1] + behind, dim, 4, DT[dt], channels_last)
    (x[:, cu[-1]:] if channels_last else x[:, :, cu[-1]:]).fill_(float("nan"))
    slots = torch.randperm(units + 3, generator=g)[:units]
    live = torch.randint(0, 2, (units,), generator=g)
    pool = normal(g, units + 3, dim, 3, dtype=DT[dt])
    pool[slots[live == 0]] = float("nan")
    if units > 2:
        slots[1], slots[2] = -1, units + 3
    before = torch.full_like(x, 7.0)
    y, bound, final = R.conv(x, w, b, pool, cu, slots, live, channels_last=channels_last, out=before)
    out, p = dev(before), dev(pool)
    got, state = xm.CausalConv1dFn(dev(x), dev(w), dev(b), p, torch.tensor(cu, dtype=index).cuda(),
                                   slots.to(index).cuda(), live.to(index).cuda(), channels_last=channels_last,
                                   output_final_state=1, out=out)
    assert got is out and state is p
    close(got, y, bound)
    assert torch.equal(torch.nan_to_num(p.cpu(), 9e4 if dt == "f32" else 9e4), torch.nan_to_num(final, 9e4))


@pytest.mark.parametrize("channels_last", [0, 1])
@pytest.mark.parametrize("inplace", [False, True])
def test_conv_given_states(xm, cuda, channels_last, inplace):
    """Row states without slots: a sequence cut in three gives the whole one's outputs, exactly."""
    g = gen(5)
    x, w, b = conv_inputs(g, 3, 300, 48, 4, torch.bfloat16, channels_last)
    whole, last = xm.CausalConv1dFn(dev(x), dev(w), dev(b), channels_last=channels_last, output_final_state=1)
    axis = 1 if channels_last else 2
    state, parts = torch.zeros(3, 48, 3, dtype=torch.bfloat16, device="cuda"), []
    for a, c in ((0, 2), (2, 129), (129, 300)):
        xi = dev(x).narrow(axis, a, c - a).contiguous()
        kw = dict(final_state=state) if inplace else {}
        part, new = xm.CausalConv1dFn(xi, dev(w), dev(b), state, channels_last=channels_last, output_final_state=1, **kw)
        assert (new is state) == inplace
        state = new
        parts.append(part)
    assert torch.equal(torch.cat(parts, axis), whole) and torch.equal(state, last)


def test_conv_infinities(xm, cuda):
    """An infinity reaches the outputs of its own window and no other."""
    g = gen(6)
    for channels_last in (0, 1):
        x, w, b = conv_inputs(g, 2, 200, 24, 4, torch.float32, channels_last)
        (x[0, 100] if channels_last else x[0, :, 100]).fill_(float("inf"))
        y, bound, _ = R.conv(x, w, b, channels_last=channels_last, silu_=False)
        close(xm.CausalConv1dFn(dev(x), dev(w), dev(b), silu=0, channels_last=channels_last), y, bound)


@pytest.mark.parametrize("channels_last", [0, 1])
def test_conv_strided_and_misaligned_inputs(xm, cuda, channels_last):
    g = gen(7)
    x, w, b = conv_inputs(g, 2, 120, 64, 4, torch.bfloat16, channels_last)
    want = xm.CausalConv1dFn(dev(x), dev(w), dev(b), channels_last=channels_last)
    wide = torch.cat([dev(x), dev(x)], 2)[..., :x.shape[2]]
    assert not wide.is_contiguous()
    assert torch.equal(xm.CausalConv1dFn(wide, dev(w), dev(b), channels_last=channels_last), want)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    flat[1:] = dev(x).flatten()
    assert torch.equal(xm.CausalConv1dFn(flat[1:].view(x.shape), dev(w), dev(b), channels_last=channels_last), want)
    o = torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")
    xm.CausalConv1dFn(dev(x), dev(w), dev(b), channels_last=channels_last, out=o[3:].view(x.shape))
    assert torch.equal(o[3:].view(x.shape), want)


# ------------------------------------------------------------------ CausalConv1dUpdateFn


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,dim,width", [(1, 1, 4), (3, 67, 4), (5, 72, 3), (2, 1024, 2), (17, 4096, 4), (1, 129, 2)])
@pytest.mark.parametrize("pool", [False, True])
def test_conv_update(xm, cuda, dt, batch, dim, width, pool):
    g = gen(batch + dim)
    x, w, b = conv_inputs(g, batch, 1, dim, width, DT[dt], 1, bias=dim != 72)
    n = batch + 4 if pool else batch
    state = normal(g, n, dim, width - 1, dtype=DT[dt])
    slots = torch.randperm(n, generator=g)[:batch] if pool else None
    if pool and batch > 2:
        slots[0], slots[1] = -1, n
    before = torch.full((batch, 1, dim), 3.0, dtype=DT[dt])
    y, bound, final = R.conv(x, w, b, state, None, slots, channels_last=True, final=state)
    if pool and batch > 2:
        y[:2], bound[:2] = 3.0, 0.0
    out, s = dev(before[:, 0]), dev(state)
    got, new = xm.CausalConv1dUpdateFn(dev(x[:, 0]), dev(w), dev(b), s, dev(slots), out=out)
    assert got is out and new is s
    close(got, y[:, 0], bound[:, 0])
    assert torch.equal(s.cpu(), final)
    if not pool:
        kept, other = dev(state), torch.empty_like(s)
        got2, new2 = xm.CausalConv1dUpdateFn(dev(x[:, 0]), dev(w), dev(b), kept, new_state=other)
        assert new2 is other and torch.equal(other, s) and torch.equal(kept.cpu(), state) and torch.equal(got2, got)


# ------------------------------------------------------------------ SelectiveScanVarlenFn


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,seqlen,dim,N,groups", [
    (1, 1, 1, 1, 1), (2, 7, 5, 3, 1), (2, 130, 64, 16, 1), (3, 257, 48, 16, 2), (1, 700, 24, 8, 1), (2, 33, 130, 17, 1),
    (1, 64, 12, 256, 3), (2, 20, 36, 128, 4), (1, 40, 260, 40, 2), (1, 100, 33, 64, 1)])
def test_scan_batched(xm, cuda, dt, batch, seqlen, dim, N, groups):
    g = gen(batch + seqlen + dim + N)
    x = scan_inputs(g, batch, seqlen, dim, N, DT[dt], groups, gate=N != 8, skip=N != 17, bias=N != 3, softplus=N != 40)
    init = normal(g, batch, dim, N) if seqlen != 130 else None
    y, bound, final, ferr = R.scan(**x, state=init, softplus=N != 40)
    got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], dev(init), delta_softplus=int(N != 40),
                                          output_final_state=1)
    close(got, y, bound)
    close(state, final, ferr)
    assert torch.equal(xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], dev(init), delta_softplus=int(N != 40)), got)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("pack", PACKS)
@pytest.mark.parametrize("dim,N", [(24, 16), (19, 5), (10, 72)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_scan_packed_pool(xm, cuda, dt, pack, dim, N, index):
    cu = PACKS[pack]
    units, behind = len(cu) - 1, 9
    g = gen(units * 17 + dim)
    x = scan_inputs(g, 1, cu[-1] + behind, dim, N, DT[dt])
    for k in ("u", "delta", "B", "C", "z"):
        x[k][:, cu[-1]:] = float("nan")
    slots = torch.randperm(units + 3, generator=g)[:units]
    live = torch.randint(0, 2, (units,), generator=g)
    pool = normal(g, units + 3, dim, N)
    pool[slots[live == 0]] = float("nan")
    if units > 2:
        slots[1], slots[2] = -1, units + 3
    before = torch.full_like(x["u"], 7.0)
    y, bound, final, ferr = R.scan(**x, state=pool, cu=cu, slots=slots, live=live, out=before)
    out, p = dev(before), dev(pool)
    got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], p, torch.tensor(cu, dtype=index).cuda(),
                                          slots.to(index).cuda(), live.to(index).cuda(), delta_softplus=1,
                                          output_final_state=1, out=out)
    assert got is out and state is p
    close(got, y, bound)
    close(p, final, ferr)


def test_scan_long_axis(xm, cuda):
    """Few channels and long sequences: the axis is split. Slow decays carry the state across the whole length."""
    g = gen(11)
    for cu, dim, N in (([0, 4096], 3, 16), ([0, 1500, 1501, 5000], 2, 4)):
        x = scan_inputs(g, 1, cu[-1], dim, N, torch.float32, softplus=False)
        x["delta"] *= 0.02
        x["A"] = -torch.rand(dim, N, generator=g)
        x["delta_bias"] = None
        init = normal(g, len(cu) - 1, dim, N)
        y, bound, final, ferr = R.scan(**x, state=init, cu=cu, softplus=False)
        got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], dev(init), torch.tensor(cu).cuda(),
                                              output_final_state=1)
        close(got, y, bound)
        close(state, final, ferr)


def test_scan_growing_states(xm, cuda):
    """A positive A lets the state grow; the decay factor is above one and the exponential unclamped."""
    g = gen(12)
    x = scan_inputs(g, 1, 60, 20, 16, torch.float32)
    x["A"] = x["A"].abs() * 0.1
    y, bound, final, ferr = R.scan(**x)
    got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], delta_softplus=1, output_final_state=1)
    close(got, y, bound)
    close(state, final, ferr)


def test_scan_extreme_steps(xm, cuda):
    """Steps from 0 to thousands (decay exactly 1 and exactly 0), and states that overflow to infinity."""
    g = gen(13)
    x = scan_inputs(g, 1, 50, 16, 16, torch.float32, softplus=False)
    x["delta"] = torch.where(torch.rand(1, 50, 16, generator=g) < 0.3, torch.zeros(()), x["delta"] * 2e4)
    x["delta_bias"] = None
    y, bound, final, ferr = R.scan(**x, softplus=False)
    got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], output_final_state=1)
    close(got, y, bound)
    close(state, final, ferr)
    x["delta"].fill_(-1e3)  # exp(dt A) overflows
    got, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], output_final_state=1)
    assert not torch.isfinite(state).any()


@pytest.mark.parametrize("inplace", [False, True])
def test_scan_given_states(xm, cuda, inplace):
    """A sequence cut in pieces continues through the states; against the definition of the whole."""
    g = gen(14)
    x = scan_inputs(g, 2, 300, 40, 16, torch.float32)
    y, bound, final, ferr = R.scan(**x)
    state, parts = torch.zeros(2, 40, 16, device="cuda"), []
    cut = lambda t, a, c: None if t is None else dev(t[:, a:c].contiguous())  # noqa: E731
    for a, c in ((0, 1), (1, 150), (150, 300)):
        kw = dict(final_state=state) if inplace else {}
        args = [cut(x[k], a, c) if x[k] is not None and x[k].dim() > 2 else dev(x[k]) for k in SCAN]
        part, new = xm.SelectiveScanVarlenFn(*args, state, delta_softplus=1, output_final_state=1, **kw)
        assert (new is state) == inplace
        state = new
        parts.append(part)
    close(torch.cat(parts, 1), y, bound)
    close(state, final, ferr)


def test_scan_matches_selective_scan_fn(xm, cuda):
    """Same values as SelectiveScanFn (channel-major, equal lengths), within both operators' bounds."""
    g = gen(15)
    x = scan_inputs(g, 2, 384, 128, 16, torch.float32)
    y, bound, final, ferr = R.scan(**x)
    t = lambda k: None if x[k] is None else dev(x[k].transpose(1, 2).contiguous())  # noqa: E731
    bc = lambda k: dev(x[k].permute(0, 2, 3, 1).contiguous())  # noqa: E731
    old, last = xm.SelectiveScanFn(t("u"), t("delta"), dev(x["A"]), bc("B"), bc("C"), dev(x["D"]), t("z"),
                                   dev(x["delta_bias"]), delta_softplus=1, apply_z_gate=1, return_last_state=1)
    new, state = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], delta_softplus=1, output_final_state=1)
    close(new, y, bound)
    scale = float(y.abs().max())
    assert float((new - old.transpose(1, 2)).abs().max()) <= 1e-4 * scale
    assert float((state - last).abs().max()) <= 1e-4 * float(final.abs().max())


def test_scan_strided_and_misaligned_inputs(xm, cuda):
    g = gen(16)
    x = scan_inputs(g, 2, 90, 64, 16, torch.bfloat16)
    want = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], delta_softplus=1)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = dev(t).flatten()
        return flat[1:].view(t.shape)

    wide = lambda t: torch.cat([dev(t), dev(t)], -1)[..., :t.shape[-1]]  # noqa: E731
    for f in (shifted, wide):
        assert torch.equal(xm.SelectiveScanVarlenFn(*[f(x[k]) for k in SCAN], delta_softplus=1), want)
    o = torch.empty(want.numel() + 3, dtype=want.dtype, device="cuda")
    xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], delta_softplus=1, out=o[3:].view(want.shape))
    assert torch.equal(o[3:].view(want.shape), want)


# ------------------------------------------------------------------ SelectiveStateUpdateFn


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,dim,N,groups", [(1, 1, 1, 1), (3, 67, 16, 1), (5, 72, 8, 2), (2, 1024, 16, 1),
                                                (4, 48, 128, 4), (2, 33, 256, 1), (3, 50, 7, 5), (2, 40, 100, 1),
                                                (70, 64, 16, 1), (1, 130, 33, 2)])
@pytest.mark.parametrize("pool", [False, True])
def test_state_update(xm, cuda, dt, batch, dim, N, groups, pool):
    g = gen(batch + dim + N)
    x = scan_inputs(g, batch, 1, dim, N, DT[dt], groups, gate=N != 8, skip=N != 7, bias=N != 128, softplus=N != 100)
    n = batch + 4 if pool else batch
    state = normal(g, n, dim, N)
    slots = torch.randperm(n, generator=g)[:batch] if pool else None
    if pool and batch > 2:
        slots[0], slots[1] = -1, n
    y, bound, final, ferr = R.scan(**x, state=state, slots=slots, softplus=N != 100, final=state)
    if pool and batch > 2:
        y[:2], bound[:2] = 3.0, 0.0
    args = [dev(x[k] if x[k] is None or x[k].dim() < 3 else x[k][:, 0]) for k in SCAN]
    out, s = torch.full((batch, dim), 3.0, dtype=DT[dt], device="cuda"), dev(state)
    got, new = xm.SelectiveStateUpdateFn(*args, s, dev(slots), delta_softplus=int(N != 100), out=out)
    assert got is out and new is s
    close(got, y[:, 0], bound[:, 0])
    close(s, final, ferr)
    if not pool:
        kept, other = dev(state), torch.empty_like(s)
        got2, new2 = xm.SelectiveStateUpdateFn(*args, kept, delta_softplus=int(N != 100), new_state=other)
        assert new2 is other and torch.equal(other, s) and torch.equal(kept.cpu(), state) and torch.equal(got2, got)


# ------------------------------------------------------------------ together, streams, graphs, sizes


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_prompt_then_tokens(xm, cuda, dt):
    """A served layer: ragged prompts through the convolution and the scan into pools of slots, then single tokens
    through the update operators with a padded batch, against the definition over the whole sequences. Between the
    convolution and the scan the reference takes the operator's own rounded output."""
    g = gen(21)
    dim, N, W, lens, steps = 96, 16, 4, [3, 1, 57, 200], 6
    total, n = sum(lens), len(lens)
    cu = [0]
    for v in lens:
        cu.append(cu[-1] + v)
    slots = torch.tensor([5, 0, 3, 6])
    xs = [normal(g, v + steps, dim, dtype=DT[dt]) for v in lens]
    w, b = (torch.rand(dim, W, generator=g) - 0.5), torch.rand(dim, generator=g) - 0.5
    p = [scan_inputs(g, 1, v + steps, dim, N, DT[dt]) for v in lens]
    for q in p[1:]:
        for k in ("A", "D", "delta_bias"):
            q[k] = p[0][k]
    conv_pool = torch.full((8, dim, W - 1), float("nan"), dtype=DT[dt], device="cuda")
    ssm_pool = torch.full((8, dim, N), float("nan"), device="cuda")
    pack = lambda parts: dev(torch.cat(parts).unsqueeze(0))  # noqa: E731
    fresh = torch.zeros(n, dtype=torch.int32, device="cuda")
    cud, sd = torch.tensor(cu, dtype=torch.int32).cuda(), slots.to(torch.int32).cuda()
    y, _ = xm.CausalConv1dFn(pack([x[:v] for x, v in zip(xs, lens)]), dev(w), dev(b), conv_pool, cud, sd, fresh,
                             channels_last=1, output_final_state=1)
    part = lambda k: pack([q[k][0, :v] for q, v in zip(p, lens)])  # noqa: E731
    out, _ = xm.SelectiveScanVarlenFn(y, part("delta"), dev(p[0]["A"]), part("B"), part("C"), dev(p[0]["D"]), part("z"),
                                      dev(p[0]["delta_bias"]), ssm_pool, cud, sd, fresh, delta_softplus=1,
                                      output_final_state=1)
    ys, outs = [y[0, a:c].cpu() for a, c in zip(cu, cu[1:])], [out[0, a:c].cpu() for a, c in zip(cu, cu[1:])]
    order = torch.cat([slots, torch.tensor([-1, -1])]).to(torch.int32).cuda()  # a padded decode batch
    row = lambda parts: dev(torch.stack(parts + [torch.full_like(parts[0], float("nan"))] * 2))  # noqa: E731
    for s in range(steps):
        y1, _ = xm.CausalConv1dUpdateFn(row([x[v + s] for x, v in zip(xs, lens)]), dev(w), dev(b), conv_pool, order)
        tok = lambda k: row([q[k][0, v + s] for q, v in zip(p, lens)])  # noqa: E731,B023
        o1, _ = xm.SelectiveStateUpdateFn(y1, tok("delta"), dev(p[0]["A"]), tok("B"), tok("C"), dev(p[0]["D"]), tok("z"),
                                          dev(p[0]["delta_bias"]), ssm_pool, order, delta_softplus=1)
        for i in range(n):
            ys[i] = torch.cat([ys[i], y1[i:i + 1].cpu()])
            outs[i] = torch.cat([outs[i], o1[i:i + 1].cpu()])
    for i in range(n):
        cy, cb, cf = R.conv(xs[i].unsqueeze(0), w, b, channels_last=True)
        close(ys[i].unsqueeze(0), cy, cb)
        assert torch.equal(conv_pool[slots[i]].cpu(), cf[0])
        q = dict(p[i], u=ys[i].unsqueeze(0))
        sy, sb, sf, se = R.scan(**q)
        close(outs[i].unsqueeze(0), sy, sb)
        close(ssm_pool[slots[i]], sf[0], se[0])
    unused = [i for i in range(8) if i not in slots.tolist()]
    assert torch.isnan(conv_pool[unused]).all() and torch.isnan(ssm_pool[unused]).all()


def _layer(xm, x, dtype, stream=None):
    y, cs = xm.CausalConv1dFn(x["x"], x["w"], None, x["cs"], x["cu"], x["slots"], channels_last=1, output_final_state=1,
                              stream=stream)
    o, ss = xm.SelectiveScanVarlenFn(y, *[x[k] for k in SCAN[1:]], x["ss"], x["cu"], x["slots"], delta_softplus=1,
                                     output_final_state=1, stream=stream)
    t, _ = xm.CausalConv1dUpdateFn(x["x"][0, :3], x["w"], None, cs, x["slots"], stream=stream)
    r, _ = xm.SelectiveStateUpdateFn(t, x["delta"][0, :3], x["A"], x["B"][0, :3], x["C"][0, :3], x["D"], x["z"][0, :3],
                                     x["delta_bias"], ss, x["slots"], delta_softplus=1, stream=stream)
    return o, r


def _layer_inputs(seed, dim=160, tokens=900):
    g = gen(seed)
    x = {k: dev(v) for k, v in scan_inputs(g, 1, tokens, dim, 16, torch.bfloat16).items()}
    x.update(x=dev(normal(g, 1, tokens, dim, dtype=torch.bfloat16)), w=torch.rand(dim, 4, generator=g).cuda(),
             cs=dev(normal(g, 5, dim, 3, dtype=torch.bfloat16)), ss=dev(normal(g, 5, dim, 16)),
             cu=torch.tensor([0, 10, 10, tokens], dtype=torch.int32).cuda(),
             slots=torch.tensor([4, 1, 2], dtype=torch.int32).cuda())
    return x


def _equal(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_two_calls_at_once(xm, cuda):
    x, y = _layer_inputs(31), _layer_inputs(32)
    want = [_layer(xm, _layer_inputs(s), torch.bfloat16) for s in (31, 32)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        x, y = _layer_inputs(31), _layer_inputs(32)
        torch.cuda.synchronize()
        a, b = _layer(xm, x, torch.bfloat16, s1), _layer(xm, y, torch.bfloat16, s2)
        torch.cuda.synchronize()
        assert _equal(a, want[0]) and _equal(b, want[1])
    with torch.cuda.stream(s1):
        x = _layer_inputs(31)
        a = _layer(xm, x, torch.bfloat16)
    torch.cuda.synchronize()
    assert _equal(a, want[0])


def test_captured_graphs(xm, cuda):
    """Two graphs of the layer, replayed in turn and at once on two streams, on inputs copied into their buffers."""
    xs = [_layer_inputs(s) for s in (33, 34)]
    want = [_layer(xm, _layer_inputs(s), torch.bfloat16) for s in (33, 34)]
    _layer(xm, _layer_inputs(33), torch.bfloat16)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_layer(xm, x, torch.bfloat16))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for order in ((0, 1), (1, 0), (0, 1)):
        for i in (0, 1):
            fresh = _layer_inputs(33 + i)
            for k in ("cs", "ss"):
                xs[i][k].copy_(fresh[k])
        torch.cuda.synchronize()
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert _equal(outs[0], want[0]) and _equal(outs[1], want[1])


def test_repeatable_bits(xm, cuda):
    a = _layer(xm, _layer_inputs(35), torch.bfloat16)
    for _ in range(3):
        assert _equal(_layer(xm, _layer_inputs(35), torch.bfloat16), a)


def test_pools_past_32_bit_offsets(xm, cuda):
    """Pools and packed rows whose element offsets pass 2^32."""
    dim, N, slots = 4096, 256, 4100  # 4.3e9 float32 state elements
    g = gen(41)
    x = scan_inputs(g, 2, 1, dim, N, torch.bfloat16)
    rows = normal(g, 2, dim, N)
    pool = torch.empty(slots, dim, N, device="cuda")
    idx = torch.tensor([slots - 1, 0], dtype=torch.int64)
    pool[idx.cuda()] = dev(rows)
    y, bound, final, ferr = R.scan(**x, state=rows)
    args = [dev(x[k] if x[k].dim() < 3 else x[k][:, 0]) for k in SCAN]
    got, _ = xm.SelectiveStateUpdateFn(*args, pool, idx.cuda(), delta_softplus=1)
    close(got, y[:, 0], bound[:, 0])
    close(pool[idx.cuda()], final, ferr)
    pool[idx.cuda()] = dev(rows)
    got, _ = xm.SelectiveScanVarlenFn(*[dev(x[k]) for k in SCAN], pool, None, idx.cuda(), delta_softplus=1,
                                      output_final_state=1)
    close(got, y, bound)
    close(pool[idx.cuda()], final, ferr)
    del pool
    # a packed row of 2^20 tokens x 4100 channels (4.3e9 elements); the sequence checked starts near its end
    tokens, dim = 1 << 20, 4100
    cu = [0, tokens - 50, tokens - 3, tokens]
    big = torch.empty(1, tokens, dim, dtype=torch.bfloat16, device="cuda")
    big[:, : tokens - 64].fill_(0.5)
    tail = normal(g, 1, 64, dim, dtype=torch.bfloat16)
    big[:, tokens - 64:] = dev(tail)
    w = torch.rand(dim, 4, generator=g) - 0.5
    cud = torch.tensor(cu, dtype=torch.int64).cuda()
    got, last = xm.CausalConv1dFn(big, dev(w), None, None, cud, channels_last=1, output_final_state=1)
    y, bound, final = R.conv(tail, w, None, cu=[14, 61, 64], channels_last=True)
    close(got[:, tokens - 50:], y[:, 14:], bound[:, 14:])
    assert torch.equal(last[1:].cpu(), final)
    del got
    q = scan_inputs(g, 1, 64, dim, 2, torch.bfloat16, gate=False)
    B = torch.zeros(1, tokens, 1, 2, dtype=torch.bfloat16, device="cuda")
    C = torch.zeros_like(B)
    B[:, tokens - 64:], C[:, tokens - 64:] = dev(q["B"]), dev(q["C"])
    q["u"] = q["delta"] = tail
    got, last = xm.SelectiveScanVarlenFn(big, big, dev(q["A"]), B, C, dev(q["D"]), None, dev(q["delta_bias"]), None, cud,
                                         delta_softplus=1, output_final_state=1)
    y, bound, final, ferr = R.scan(**q, cu=[14, 61, 64])
    close(got[:, tokens - 50:], y[:, 14:], bound[:, 14:])
    close(last[1:], final, ferr)


@pytest.mark.parametrize("channels_last", [0, 1])
def test_more_sequences_than_a_grid_dimension(xm, cuda, channels_last):
    """70001 sequences of one call equal the same ones in several calls, bit by bit."""
    g = gen(61)
    n, dim = 70001, 8
    cuts = [(0, 30000), (30000, 65536), (65536, n)]
    x, w, b = conv_inputs(g, n, 3, dim, 4, torch.bfloat16, channels_last)
    x, w, b = dev(x), dev(w), dev(b)
    y, last = xm.CausalConv1dFn(x, w, b, channels_last=channels_last, output_final_state=1)
    parts = [xm.CausalConv1dFn(x[a:c], w, b, channels_last=channels_last, output_final_state=1) for a, c in cuts]
    assert torch.equal(torch.cat([p[0] for p in parts]), y) and torch.equal(torch.cat([p[1] for p in parts]), last)
    if not channels_last:
        return
    q = {k: dev(v) for k, v in scan_inputs(g, n, 3, dim, 16, torch.bfloat16).items()}
    cut = lambda t, a, c: t[a:c] if t.dim() > 2 else t  # noqa: E731
    y, last = xm.SelectiveScanVarlenFn(*[q[k] for k in SCAN], delta_softplus=1, output_final_state=1)
    parts = [xm.SelectiveScanVarlenFn(*[cut(q[k], a, c) for k in SCAN], delta_softplus=1, output_final_state=1)
             for a, c in cuts]
    assert torch.equal(torch.cat([p[0] for p in parts]), y) and torch.equal(torch.cat([p[1] for p in parts]), last)
    state = torch.randn(n, dim, 16, device="cuda")
    tok = lambda t, a, c: t[a:c, 0].contiguous() if t.dim() > 2 else t  # noqa: E731
    parts = [xm.SelectiveStateUpdateFn(*[tok(q[k], a, c) for k in SCAN], state[a:c].clone(), delta_softplus=1)
             for a, c in cuts]
    y, state = xm.SelectiveStateUpdateFn(*[tok(q[k], 0, n) for k in SCAN], state, delta_softplus=1)
    assert torch.equal(torch.cat([p[0] for p in parts]), y) and torch.equal(torch.cat([p[1] for p in parts]), state)
    cs = last_inputs = torch.randn(n, dim, 3, device="cuda").to(torch.bfloat16)
    parts = [xm.CausalConv1dUpdateFn(x[a:c, 0].contiguous(), w, b, cs[a:c].clone()) for a, c in cuts]
    y, cs = xm.CausalConv1dUpdateFn(x[:, 0].contiguous(), w, b, cs)
    assert cs is last_inputs
    assert torch.equal(torch.cat([p[0] for p in parts]), y) and torch.equal(torch.cat([p[1] for p in parts]), cs)
    # packed: as many sequences, some empty, over one row
    lens = torch.randint(0, 4, (n,), generator=g)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    total = int(cu[-1])
    flat = x.reshape(1, -1, dim)[:, :total].contiguous()
    y, last = xm.CausalConv1dFn(flat, w, b, None, cu.cuda(), channels_last=1, output_final_state=1)
    half = int(cu[40000])
    a = xm.CausalConv1dFn(flat[:, :half], w, b, None, cu[:40001].cuda(), channels_last=1, output_final_state=1)
    c = xm.CausalConv1dFn(flat[:, half:], w, b, None, (cu[40000:] - half).cuda(), channels_last=1, output_final_state=1)
    assert torch.equal(torch.cat([a[0], c[0]], 1), y) and torch.equal(torch.cat([a[1], c[1]]), last)


def test_a_slot_named_twice_touches_nothing_else(xm, cuda):
    x = _layer_inputs(62)
    before = {k: x[k].clone() for k in ("cs", "ss")}
    x["slots"] = torch.tensor([3, 3, 1], dtype=torch.int32).cuda()
    _layer(xm, x, torch.bfloat16)
    for k in ("cs", "ss"):
        for i in (0, 2, 4):
            assert torch.equal(x[k][i], before[k][i])
        assert torch.isfinite(x[k].float()).all()


def test_refusals_on_the_device(xm, cuda):
    """What only a device tensor can show: strided states in place, host tensors among device ones, strided outputs."""
    g = gen(63)
    x, w, b = conv_inputs(g, 4, 6, 16, 4, torch.float32, 1)
    x, w, b = dev(x), dev(w), dev(b)
    wide = torch.zeros(4, 16, 6, device="cuda")
    with pytest.raises(xm.XmError, match="state is updated in place and must be contiguous"):
        xm.CausalConv1dUpdateFn(x[:, 0].contiguous(), w, b, wide[..., :3])
    with pytest.raises(xm.XmError, match="initial_state is updated in place and must be contiguous"):
        xm.CausalConv1dFn(x, w, b, wide[..., :3], None, torch.arange(4, device="cuda"), channels_last=1,
                          output_final_state=1)
    with pytest.raises(xm.XmError, match="weight must be a tensor on cuda:0"):
        xm.CausalConv1dFn(x, w.cpu(), b, channels_last=1)
    with pytest.raises(xm.XmError, match="out must be a contiguous tensor on cuda:0"):
        xm.CausalConv1dFn(x, w, b, channels_last=1, out=torch.empty(4, 6, 32, device="cuda")[..., :16])
    with pytest.raises(xm.XmError, match="an output must not overlap an input"):
        xm.CausalConv1dFn(x, w, b, channels_last=1, out=x)
    with pytest.raises(xm.XmError, match="the state output must be a contiguous tensor on cuda:0"):
        xm.CausalConv1dUpdateFn(x[:, 0].contiguous(), w, b, wide[..., :3].contiguous(), new_state=wide[..., :3])
    with pytest.raises(xm.XmError, match="has_initial_state must be int32 or int64"):
        xm.CausalConv1dFn(x, w, b, torch.zeros(4, 16, 3, device="cuda"), None, None,
                          torch.ones(4, dtype=torch.bool, device="cuda"), channels_last=1)
    # a strided input state is copied where it is not written
    got, new = xm.CausalConv1dFn(x, w, b, wide[..., :3], channels_last=1, output_final_state=1)
    assert torch.equal(got, xm.CausalConv1dFn(x, w, b, channels_last=1)) and not torch.equal(new, wide[..., :3])


def test_malformed_offsets_stay_inside(xm, cuda):
    """Offsets that descend or leave the row address nothing outside it (values are not defined)."""
    x = _layer_inputs(51)
    pad = torch.full((1, 64, 160), 5.0, dtype=torch.bfloat16, device="cuda")
    for cu in ([-5, 20, 10, 100000], [900, 900, 900, 900], [2**31 - 1, -2**31, 0, 7]):
        x["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
        out = torch.cat([pad, torch.zeros(1, 900, 160, dtype=torch.bfloat16, device="cuda"), pad], 1)
        mid = out[:, 64:964]
        xm.CausalConv1dFn(x["x"], x["w"], None, x["cs"], x["cu"], x["slots"], channels_last=1, output_final_state=1, out=mid)
        xm.SelectiveScanVarlenFn(*[x[k] for k in SCAN], x["ss"], x["cu"], x["slots"], delta_softplus=1,
                                 output_final_state=1, out=mid)
        cf = x["x"].transpose(1, 2).contiguous()
        xm.CausalConv1dFn(cf, x["w"], None, x["cs"], x["cu"], x["slots"], output_final_state=1)
        torch.cuda.synchronize()
        assert bool((out[:, :64] == 5).all()) and bool((out[:, 964:] == 5).all())
