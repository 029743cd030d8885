"""Edges of the gated recurrence on the GPU: gates shut on purpose, whose small
shares decide the result. Definitions and error bounds: recurrence_reference.py."""

from __future__ import annotations

import pytest
import torch

import recurrence_reference as Q
from test_recurrence_gpu import DT, close, dev, gen, normal

pytestmark = pytest.mark.gpu

LOGITS = torch.tensor([-60.0, -70.0, -87.0, -200.0])
BOUNDS = torch.tensor([0.999, 0.99999, 1 - 2.0**-24, 0.0])
# one of each way that a call is cut: a warp to a row, a block to a row, segments in two kernels, blocks whose warps take
# turns (of eight and of four)
CUTS = [(2, 40, 70), (1, 700, 70), (1, 2600, 70), (8, 256, 1280), (8, 256, 2560)]


def shut(g, batch, seqlen, dim, dtype):
    """Gates that keep next to nothing of their own, in channels whose lower bounds keep all but a little: from a state of
    zero, what is taken up is the whole result."""
    x = normal(g, batch, seqlen, dim, dtype=dtype)
    f = LOGITS[torch.randint(0, 4, (batch, seqlen, dim), generator=g)].to(dtype)
    return x, f, BOUNDS[torch.arange(dim) % 4].contiguous()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,seqlen,dim", CUTS)
def test_shut_gates(xm, cuda, dt, batch, seqlen, dim):
    """The share taken up, (1 - lower bound) sigmoid(-f), keeps its relative precision however far f is below zero."""
    g = gen(71)
    x, f, low = shut(g, batch, seqlen, dim, DT[dt])
    y, bound, final, fb = Q.recurrence(x, f, low)
    got, last = xm.GatedRecurrenceFn(dev(x), dev(f), dev(low), output_final_state=1)
    close(got, y, bound)
    close(last, final, fb)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,dim", [(3, 72), (3, 67), (500, 1024)])
def test_shut_gates_of_single_tokens(xm, cuda, dt, batch, dim):
    g = gen(72)
    x, f, low = shut(g, batch, 1, dim, DT[dt])
    y, bound, final, fb = Q.recurrence(x, f, low)
    got, state = xm.GatedRecurrenceUpdateFn(dev(x[:, 0]), dev(f[:, 0]), dev(low), torch.zeros(batch, dim, device="cuda"))
    close(got, y[:, 0], bound[:, 0])
    close(state, final, fb)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("batch,seqlen,dim", CUTS)
@pytest.mark.parametrize("scale", [1.0, 2.0**-80])
def test_shut_gates_backward(xm, cuda, dt, batch, seqlen, dim, scale):
    """The lower bounds' gradient is sum G (h - x) sigmoid(-f) whatever the bounds are, 1 among them, and however small G
    is; behind a bound of 1 the inputs have none."""
    g = gen(73)
    x, f, low = shut(g, batch, seqlen, dim, DT[dt])
    low[low == 0] = 1.0
    y = Q.recurrence(x, f, low)[0].to(DT[dt])
    dy = normal(g, batch, seqlen, dim, std=scale).to(DT[dt])  # (2^-80 is below float16's range: zero)
    want = Q.recurrence_grad(dy, x, f, y, low)
    got = xm.GatedRecurrenceGradFn(dev(dy), dev(x), dev(f), dev(y), dev(low))
    for k in range(3):
        close(got[k], *want[k])
    assert not bool(got[0][..., low == 1].any()) and not bool(got[1][..., low == 1].any())


def shut_behind_a_group(dim, tokens=256, batch=8):
    """Gates open for a while, then shut: products of gates that leave float32's range meet states that have not."""
    f = torch.full((batch, tokens, dim), 30.0)
    f[:, 40:200] = -30.0
    return torch.zeros(batch, tokens, dim), f


@pytest.mark.parametrize("dim", [1280, 2560])
def test_channels_do_not_touch_each_other(xm, cuda, dim):
    """Nor do sequences: an infinite channel leaves every bit of the others as it is, forward and backward."""
    x, f = (dev(t) for t in shut_behind_a_group(dim))
    ones = torch.ones(8, dim, device="cuda")
    odd = ones.clone()
    odd[::2, ::7] = float("inf")
    odd[1, 3] = float("nan")
    same = odd == ones
    y, last = xm.GatedRecurrenceFn(x, f, None, ones, output_final_state=1)
    y2, last2 = xm.GatedRecurrenceFn(x, f, None, odd, output_final_state=1)
    rows = same[:, None].expand_as(y)
    assert torch.equal(y[rows], y2[rows]) and torch.equal(last[same], last2[same])
    assert bool(torch.isinf(y2[0, :, 0]).all())
    got = xm.GatedRecurrenceGradFn(x, x, f, y, None, ones, None, ones)
    got2 = xm.GatedRecurrenceGradFn(x, x, f, y, None, ones, None, odd)
    assert all(torch.equal(a[rows], b[rows]) for a, b in zip(got[:2], got2[:2]))
    assert torch.equal(got[3][same], got2[3][same])


@pytest.mark.parametrize("dim", [1250, 1251])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_bits_do_not_depend_on_what_ran_before(xm, cuda, dt, dim):
    """Channels that are not there are not looked at: shared memory still holds what a kernel before left in their place."""
    x, f = (dev(t).to(DT[dt]) for t in shut_behind_a_group(dim))
    ones = torch.ones(8, dim, device="cuda")
    y = xm.GatedRecurrenceFn(x, f, None, ones)
    results = []
    for fill in (0.0, float("inf"), float("nan")):
        before = torch.full((8, 256, 2560), fill, dtype=DT[dt], device="cuda")
        xm.GatedRecurrenceFn(before, before)
        forward = xm.GatedRecurrenceFn(x, f, None, ones, output_final_state=1)
        xm.GatedRecurrenceGradFn(before, before, before, before)
        results.append((*forward, *xm.GatedRecurrenceGradFn(x, x, f, y, None, ones, None, ones)))
    for r in results[1:]:
        assert all(a is b or torch.equal(a, b) for a, b in zip(r, results[0]))
