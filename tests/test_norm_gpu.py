"""LayerNormFn and LayerNormGradFn on the GPU against their float64 definitions
(recurrence_reference.py, which also gives the error bounds)."""

from __future__ import annotations

import pytest
import torch

import recurrence_reference as Q
from test_recurrence_gpu import DT, close, dev, gen, normal

pytestmark = pytest.mark.gpu

SHAPES = [((1,), 1), ((3,), 2), ((2, 5), 7), ((4,), 8), ((1, 1, 3), 64), ((33,), 100), ((7,), 128), ((1,), 1000),
          ((300,), 72), ((9,), 1024), ((5,), 1025), ((2,), 2048), ((3,), 4096), ((1,), 4096), ((2,), 5003), ((4,), 8192),
          ((2,), 16384), ((2,), 16392), ((1,), 40000), ((2,), 100003), ((), 96),
          ((5,), 362), ((4,), 1026), ((3,), 2050), ((2,), 4098), ((2,), 8194)]


def rows(g, lead, dim, dtype):
    """Channels of different scale and offset."""
    return (normal(g, *lead, dim) * torch.exp(normal(g, dim, std=0.5)) + normal(g, dim, std=0.5)).to(dtype)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lead,dim", SHAPES)
@pytest.mark.parametrize("rms,residual", [(0, True), (1, True), (0, False), (1, False)])
def test_norm(xm, cuda, dt, lead, dim, rms, residual):
    g = gen(dim + rms)
    x = rows(g, lead, dim, DT[dt])
    w = normal(g, dim, std=0.3, mean=1.0) if dim != 100 else None
    b = normal(g, dim) if dim % 3 != 1 else None
    r = normal(g, *lead, dim, dtype=DT[dt], std=2.0) if residual else None
    eps = 1e-5 if dim != 64 else 0.01
    (y, yb), (s, sb), (st, stb) = Q.norm(x, w, b, r, eps, bool(rms))
    got = xm.LayerNormFn(dev(x), dev(w), dev(b), dev(r), eps=eps, rms=rms, output_stats=1)
    close(got[0], y, yb)
    close(got[-1], st, stb)
    if residual:
        close(got[1], s, sb)
    plain = xm.LayerNormFn(dev(x), dev(w), dev(b), dev(r), eps=eps, rms=rms)
    assert torch.equal(plain[0] if residual else plain, got[0])
    if residual:  # the residual stream in place
        stream = dev(r)
        got2 = xm.LayerNormFn(dev(x), dev(w), dev(b), stream, eps=eps, rms=rms, residual_out=stream)
        assert got2[1] is stream and torch.equal(stream, got[1]) and torch.equal(got2[0], got[0])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lead,dim", SHAPES + [((1200,), 40), ((700,), 1000), ((513,), 67)])
@pytest.mark.parametrize("rms,residual,bias", [(0, True, 1), (1, False, 0), (0, False, 1), (1, True, 0)])
def test_norm_grad(xm, cuda, dt, lead, dim, rms, residual, bias):
    g = gen(dim + rms + 5)
    x, dy = rows(g, lead, dim, DT[dt]), normal(g, *lead, dim, dtype=DT[dt])
    w = normal(g, dim, std=0.3, mean=1.0) if dim != 100 else None
    r = normal(g, *lead, dim, dtype=DT[dt]) if residual else None
    st = Q.norm(x, None, None, None, 1e-5, bool(rms))[2][0].float()
    want = Q.norm_grad(dy, x, w, st, r, bool(rms))
    got = xm.LayerNormGradFn(dev(dy), dev(x), dev(w), dev(st), dev(r), rms=rms, output_bias_grad=bias)
    close(got[0], *want[0])
    assert (got[1] is None) == (w is None) and (got[2] is None) == (not bias)
    if w is not None:
        close(got[1], *want[1])
    if bias:
        close(got[2], *want[2])
    again = xm.LayerNormGradFn(dev(dy), dev(x), dev(w), dev(st), dev(r), rms=rms, output_bias_grad=bias)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, again))


def test_rows_with_a_large_mean(xm, cuda):
    """The variance of rows far from zero survives: it is taken of the differences."""
    g = gen(3)
    x = normal(g, 6, 1000, std=0.5, mean=3000.0)
    (y, yb), _, (st, stb) = Q.norm(x)
    got, stats = xm.LayerNormFn(dev(x), output_stats=1)
    close(got, y, yb)
    close(stats, st, stb)
    assert float((got.cpu() - y).abs().max()) < 0.01


def test_constant_and_zero_rows(xm, cuda):
    """No variance: the differences are zero, y is the bias; eps keeps rstd finite."""
    b = torch.rand(520)
    for value in (0.0, 2.5):
        x = torch.full((3, 520), value)
        for dtype in DT.values():
            y, st = xm.LayerNormFn(x.to(dtype).cuda(), None, dev(b), output_stats=1)
            assert torch.equal(y.cpu(), b.to(dtype).expand(3, 520))
            assert torch.equal(st[:, 0].cpu(), torch.full((3,), value))
            assert torch.allclose(st[:, 1].cpu(), torch.tensor(1e-5).rsqrt().expand(3), rtol=1e-6)


def test_infinities_and_nan_stay_in_their_row(xm, cuda):
    g = gen(4)
    for dim in (96, 4096, 20000):
        x = normal(g, 5, dim)
        x[1, 7], x[3, 0] = float("inf"), float("nan")
        w, b = normal(g, dim), normal(g, dim)
        (y, yb), _, _ = Q.norm(x[::2], w, b)
        got = xm.LayerNormFn(dev(x), dev(w), dev(b))
        close(got[::2], y, yb)
        assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[3]).all())
        st = Q.norm(x[::2])[2][0].float()
        full = torch.zeros(5, 2)
        full[::2] = st
        dy = normal(g, 5, dim)
        want = Q.norm_grad(dy[::2], x[::2], w, st)
        dx, dw, _ = xm.LayerNormGradFn(dev(dy), dev(x), dev(w), dev(full))
        close(dx[::2], *want[0])
        assert bool(torch.isnan(dw[7])) and bool(torch.isnan(dw[0])) and not bool(torch.isnan(dw[8]))


def test_strided_and_misaligned(xm, cuda):
    g = gen(5)
    for dtype in DT.values():
        for dim in (64, 1000, 4096):
            x, r, w, b = rows(g, (4,), dim, dtype), normal(g, 4, dim, dtype=dtype), normal(g, dim), normal(g, dim)
            dy = normal(g, 4, dim, dtype=dtype)
            (y, yb), (s, sb), (st, stb) = Q.norm(x, w, b, r)
            grads = Q.norm_grad(dy, s.to(dtype), w, st.float(), r)
            for off in (1, 2, 3, 4):
                place = lambda t: torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape)  # noqa: E731
                moved = [place(t) for t in (x, w, b, r, dy)]
                for d, src in zip(moved, (x, w, b, r, dy)):
                    d.copy_(src)
                outs = dict(out=place(x), residual_out=place(r), stats=place(st.float()))
                got = xm.LayerNormFn(*moved[:4], output_stats=1, **outs)
                assert got[0] is outs["out"] and got[1] is outs["residual_out"] and got[2] is outs["stats"]
                close(got[0], y, yb)
                close(got[1], s, sb)
                close(got[2], st, stb)
                sums, stats = place(x), place(st.float())
                sums.copy_(s.to(dtype))
                stats.copy_(st.float())
                gouts = (place(x), place(w), place(b))
                got = xm.LayerNormGradFn(moved[4], sums, moved[1], stats, moved[3], output_bias_grad=1, out=gouts)
                for k in range(3):
                    assert got[k] is gouts[k]
                    close(got[k], *grads[k])
            wide = torch.cat([dev(x), dev(x)], 1)[:, :dim]
            assert torch.equal(xm.LayerNormFn(wide, dev(w)), xm.LayerNormFn(dev(x), dev(w)))


def test_a_row_does_not_depend_on_its_batch(xm, cuda):
    g = gen(6)
    for dim in (40, 512, 4096, 9000):
        x, w = dev(rows(g, (900,), dim, torch.bfloat16)), dev(normal(g, dim))
        y = xm.LayerNormFn(x, w)
        for part in (slice(0, 1), slice(3, 40), slice(899, 900)):
            assert torch.equal(xm.LayerNormFn(x[part], w), y[part])


def test_empty_calls(xm, cuda):
    x, w, b = torch.empty(0, 24, device="cuda"), torch.rand(24, device="cuda"), torch.rand(24, device="cuda")
    assert xm.LayerNormFn(x, w, b).shape == (0, 24)
    y, s, st = xm.LayerNormFn(x, w, b, x.clone(), output_stats=1)
    assert y.shape == s.shape == (0, 24) and st.shape == (0, 2)
    dx, dw, db = xm.LayerNormGradFn(x, x, w, torch.empty(0, 2, device="cuda"), output_bias_grad=1)
    assert dx.shape == (0, 24) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_many_rows_and_offsets_past_32_bits(xm, cuda):
    """More than 2^31 elements: the last rows, and the weights' gradient over all of them."""
    n, dim = 2**19 + 3, 4096
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda")
    g = gen(7)
    at = [0, 2**18, 2**19 - 1, 2**19, n - 1]
    some, w, b = rows(g, (5,), dim, torch.bfloat16), normal(g, dim), normal(g, dim)
    x[torch.tensor(at).cuda()] = some.cuda()
    (y, yb), _, (st, stb) = Q.norm(some, w, b)
    got, stats = xm.LayerNormFn(x, dev(w), dev(b), output_stats=1)
    close(got[torch.tensor(at).cuda()], y, yb)
    close(stats[torch.tensor(at).cuda()], st, stb)
    assert torch.equal(got[5], dev(b).to(torch.bfloat16)) and torch.equal(got[2**19 + 1], got[5])
    del got
    dys = normal(g, 5, dim, dtype=torch.bfloat16)
    want = Q.norm_grad(dys, some, w, stats[torch.tensor(at).cuda()].cpu())
    dy = torch.zeros_like(x)
    dy[torch.tensor(at).cuda()] = dys.cuda()
    dx, dw, db = xm.LayerNormGradFn(dy, x, dev(w), stats, output_bias_grad=1)
    close(dx[torch.tensor(at).cuda()], *want[0])
    close(dw, *want[1])
    close(db, *want[2])


def test_more_rows_than_a_grid_dimension(xm, cuda):
    n, dim = 200003, 5
    g = gen(8)
    x, w, dy = normal(g, n, dim), normal(g, dim), normal(g, n, dim)
    (y, yb), _, (st, stb) = Q.norm(x, w)
    got, stats = xm.LayerNormFn(dev(x), dev(w), output_stats=1)
    close(got, y, yb)
    close(stats, st, stb)
    want = Q.norm_grad(dy, x, w, stats.cpu())
    res = xm.LayerNormGradFn(dev(dy), dev(x), dev(w), stats, output_bias_grad=1)
    for k in range(3):
        close(res[k], *want[k])


def test_refusals_on_the_device(xm, cuda):
    from types import SimpleNamespace

    x, w, st = torch.rand(4, 8, device="cuda"), torch.rand(8, device="cuda"), torch.rand(4, 2, device="cuda")
    other = SimpleNamespace(device_index=1, cuda_stream=torch.cuda.default_stream(0).cuda_stream)
    wide = torch.rand(4, 16, device="cuda")[:, :8]
    fn, grad = xm.LayerNormFn, xm.LayerNormGradFn
    for call, match in (
        (lambda: fn(x, w.cpu()), "weight must be a tensor on cuda:0"),
        (lambda: fn(x, w.half()), "float32"),
        (lambda: fn(x, w, eps=-1.0), "eps"),
        (lambda: fn(x, w, None, x.half()), "float32"),
        (lambda: fn(x, w, None, x[:2]), "residual shape must match x"),
        (lambda: fn(x, out=x), "an output must not overlap an input"),
        (lambda: fn(x, w, None, x.clone(), residual_out=x), "an output must not overlap an input"),
        (lambda: fn(x, w, None, wide, residual_out=wide), "updated in place and must be contiguous"),
        (lambda: fn(x, w, stream=other), "stream belongs to another device"),
        (lambda: fn(x, w, output_stats=1, stats=torch.empty(4, 3, device="cuda")), "stats must be float32 with shape"),
        (lambda: grad(x, x, w, st[:3]), "stats must have"),
        (lambda: grad(x, x.half(), w, st), "float32"),
        (lambda: grad(x, x, w, st, out=(x, None, None)), "an output must not overlap an input"),
        (lambda: grad(x, x, w, st, stream=other), "stream belongs to another device"),
        (lambda: grad(x, x, w, st.half()), "float32"),
    ):
        with pytest.raises(xm.XmError, match=match):
            call()
