"""The gated linear recurrence and layer norm without a GPU: attribute defaults,
shape and workspace queries, what each refuses, and their float64 definitions
against autograd and differences."""

from __future__ import annotations

import ctypes

import pytest
import torch

import recurrence_reference as Q
import test_serving_cpu as C

F32, I32, I64, F16, BF16 = C.F32, C.I32, C.I64, C.F16, C.BF16


def gate_in(m, io=BF16, x=(2, 16, 8), f=None, bound=(8,), init=(0,), cu=(0,), slots=(0,), live=(0,)):
    return [m(x, io), m(f or x, io), m(bound), m(init), m(cu, I32), m(slots, I64), m(live, I32)]


def grad_in(m, io=BF16, dy=(2, 16, 8), x=None, f=None, y=None, bound=(8,), init=(0,), cu=(0,), dlast=(0,)):
    return [m(dy, io), m(x or dy, io), m(f or dy, io), m(y or dy, io), m(bound), m(init), m(cu, I32), m(dlast)]


def update_in(m, io=BF16, x=(3, 8), f=None, bound=(8,), state=(3, 8), slots=(0,)):
    return [m(x, io), m(f or x, io), m(bound), m(state), m(slots, I32)]


def norm_in(m, io=BF16, x=(2, 5, 8), weight=(8,), bias=(8,), res=(0,)):
    return [m(x, io), m(weight), m(bias), m(res, io)]


def norm_grad_in(m, io=BF16, dy=(2, 5, 8), x=None, weight=(8,), stats=(2, 5, 2), dres=(0,)):
    return [m(dy, io), m(x or dy, io), m(weight), m(stats), m(dres, io)]


MAKE = dict(gated_recurrence=gate_in, gated_recurrence_grad=grad_in, gated_recurrence_update=update_in,
            layer_norm=norm_in, layer_norm_grad=norm_grad_in)


def attrs_of(xm, op, *values):
    kind = dict(gated_recurrence=xm.GatedRecurrenceAttrs, gated_recurrence_grad=xm.GatedRecurrenceGradAttrs,
                gated_recurrence_update=xm.GatedRecurrenceUpdateAttrs, layer_norm=xm.LayerNormAttrs,
                layer_norm_grad=xm.LayerNormGradAttrs)[op]
    a = kind()
    getattr(xm.load_library(), f"xm_{op}_attrs_default")(ctypes.byref(a))
    for (name, _), v in zip(kind._fields_, values):
        setattr(a, name, v)
    return a


def test_attribute_defaults(xm):
    lib = xm.load_library()
    want = dict(gated_recurrence=(0,), gated_recurrence_grad=(0, 0), gated_recurrence_update=(0,),
                layer_norm=(pytest.approx(1e-5), 0, 0), layer_norm_grad=(0, 0))
    for op, values in want.items():
        a = attrs_of(xm, op)
        assert tuple(getattr(a, n) for n, _ in a._fields_) == values
        assert getattr(lib, f"xm_{op}_check_attrs")(ctypes.byref(a)) == 0
        assert getattr(lib, f"xm_{op}_check_attrs")(None) == xm.XM_ERR_INVALID_ARGUMENT
    for eps in (float("nan"), float("inf"), -1e-5):
        assert lib.xm_layer_norm_check_attrs(ctypes.byref(attrs_of(xm, "layer_norm", eps))) == xm.XM_ERR_INVALID_ARGUMENT
        assert lib.xm_last_error().decode() == "LayerNormFn requires a finite eps of at least 0"
    assert lib.xm_layer_norm_check_attrs(ctypes.byref(attrs_of(xm, "layer_norm", 0.0))) == 0
    assert lib.xm_gated_recurrence_update_check_attrs(ctypes.byref(attrs_of(xm, "gated_recurrence_update", 1))) != 0
    assert {"GatedRecurrenceFn", "GatedRecurrenceGradFn", "GatedRecurrenceUpdateFn", "LayerNormFn",
            "LayerNormGradFn"} <= set(xm.OP_NAMES) & set(xm.__all__)


def test_valid_shapes(xm):
    m = C.Maker(xm)
    ok = lambda op, tensors, *attrs: C.shape_query(xm, op, attrs_of(xm, op, *attrs), tensors)[::2]  # noqa: E731
    for io in (F32, BF16, F16):
        assert ok("gated_recurrence", gate_in(m, io)) == (0, (2, 16, 8))
        assert ok("gated_recurrence", gate_in(m, io, bound=(0,), init=(2, 8)), 1) == (0, (2, 16, 8))
        assert ok("gated_recurrence_grad", grad_in(m, io, init=(2, 8), dlast=(2, 8)), 1, 1) == (0, (2, 16, 8))
        assert ok("gated_recurrence_update", update_in(m, io)) == (0, (3, 8))
        assert ok("layer_norm", norm_in(m, io, res=(2, 5, 8))) == (0, (2, 5, 8))
        assert ok("layer_norm", norm_in(m, io, x=(8,), weight=(0,), bias=(0,))) == (0, (8,))
        assert ok("layer_norm_grad", norm_grad_in(m, io, weight=(0,))) == (0, (2, 5, 8))
    assert ok("gated_recurrence", gate_in(m, x=(1, 16, 8), cu=(4,), init=(9, 8), slots=(3,), live=(3,)), 1) == (0, (1, 16, 8))
    assert ok("gated_recurrence", gate_in(m, x=(0, 16, 8), init=(64, 8))) == (0, (0, 16, 8))
    assert ok("gated_recurrence", gate_in(m, x=(2, 0, 8))) == (0, (2, 0, 8))
    assert ok("gated_recurrence_grad", grad_in(m, dy=(1, 16, 8), cu=(4,), init=(3, 8), dlast=(3, 8))) == (0, (1, 16, 8))
    assert ok("layer_norm", norm_in(m, x=(0, 8))) == (0, (0, 8))
    assert ok("layer_norm_grad", norm_grad_in(m, dy=(0, 8), stats=(0, 2))) == (0, (0, 8))


REFUSED = [
    ("gated_recurrence", dict(x=(16, 8)), "x must have rank 3"),
    ("gated_recurrence", dict(f=(2, 16, 7)), "f shape must match x"),
    ("gated_recurrence", dict(bound=(7,)), "lower_bound must be empty or have shape (dim)"),
    ("gated_recurrence", dict(init=(2, 9)), "initial_state must have shape (sequences, dim)"),
    ("gated_recurrence", dict(init=(3, 8)), "initial_state must have shape (sequences, dim)"),
    ("gated_recurrence", dict(init=(3, 8, 1)), "initial_state must have shape (sequences, dim)"),
    ("gated_recurrence", dict(init=(5, 9), slots=(2,)), "initial_state must have shape (slots, dim)"),
    ("gated_recurrence", dict(slots=(2,)), "state_indices needs a non-empty initial_state"),
    ("gated_recurrence", dict(init=(5, 8), slots=(3,)), "state_indices must be empty or have one element per sequence"),
    ("gated_recurrence", dict(live=(3,)), "has_initial_state must be empty or have one element per sequence"),
    ("gated_recurrence", dict(cu=(3,)), "GatedRecurrenceFn with cu_seqlens expects batch 1"),
    ("gated_recurrence", dict(x=(1, 16, 8), cu=(1,)), "cu_seqlens must be 1-D with at least 2 offsets"),
    ("gated_recurrence", dict(x=(70000, 40000, 8)), "GatedRecurrenceFn of 2^31 - 4096 tokens or more is not supported"),
    ("gated_recurrence", dict(x=(1, 2, (1 << 30) + 1), bound=(0,)), "dim above 2^30 is not supported"),
    ("gated_recurrence", dict(x=(2, 8, -1)), "x has a negative dimension"),
    ("gated_recurrence", dict(x=(1 << 30, 1 << 30, 1 << 30)), "x has too many elements"),
    ("gated_recurrence_grad", dict(dy=(16, 8)), "dy must have rank 3"),
    ("gated_recurrence_grad", dict(x=(2, 16, 7)), "x shape must match dy"),
    ("gated_recurrence_grad", dict(f=(2, 15, 8)), "f shape must match dy"),
    ("gated_recurrence_grad", dict(y=(1, 16, 8)), "y shape must match dy"),
    ("gated_recurrence_grad", dict(bound=(9,)), "lower_bound must be empty or have shape (dim)"),
    ("gated_recurrence_grad", dict(bound=(0,)), "output_lower_bound_grad requires a non-empty lower_bound"),
    ("gated_recurrence_grad", dict(init=(3, 8)), "initial_state must have shape (sequences, dim)"),
    ("gated_recurrence_grad", dict(dlast=(3, 8)), "d_final_state must have shape (sequences, dim)"),
    ("gated_recurrence_grad", dict(cu=(3,)), "GatedRecurrenceGradFn with cu_seqlens expects batch 1"),
    ("gated_recurrence_update", dict(x=(3, 8, 1)), "x must have rank 2"),
    ("gated_recurrence_update", dict(state=(2, 8)), "state must have shape (sequences, dim)"),
    ("gated_recurrence_update", dict(state=(0,)), "GatedRecurrenceUpdateFn needs a non-empty state"),
    ("layer_norm", dict(x=()), "x must have at least one axis"),
    ("layer_norm", dict(weight=(7,)), "weight must be empty or have shape (dim)"),
    ("layer_norm", dict(weight=(1, 8)), "weight must be empty or have shape (dim)"),
    ("layer_norm", dict(bias=(9,)), "bias must be empty or have shape (dim)"),
    ("layer_norm", dict(res=(2, 5, 7)), "residual shape must match x"),
    ("layer_norm", dict(x=(1, (1 << 30) + 1), weight=(0,), bias=(0,)), "dim above 2^30 is not supported"),
    ("layer_norm", dict(x=(1 << 16, 1 << 15, 8)), "LayerNormFn of 2^31 rows or more is not supported"),
    ("layer_norm_grad", dict(x=(2, 5, 7)), "x shape must match dy"),
    ("layer_norm_grad", dict(weight=(9,)), "weight must be empty or have shape (dim)"),
    ("layer_norm_grad", dict(stats=(2, 5, 3)), "stats must have x's leading axes and a last one of 2 (mean, rstd)"),
    ("layer_norm_grad", dict(stats=(0,)), "stats must have x's leading axes and a last one of 2 (mean, rstd)"),
    ("layer_norm_grad", dict(dres=(2, 4, 8)), "d_residual shape must match dy"),
]


def default_attrs(xm, op):
    return attrs_of(xm, op, 1, 1) if op == "gated_recurrence_grad" else attrs_of(xm, op)


@pytest.mark.parametrize("op,change,message", REFUSED)
def test_refused_inputs(xm, op, change, message):
    tensors = MAKE[op](C.Maker(xm), **change)
    rc, msg, _ = C.shape_query(xm, op, default_attrs(xm, op), tensors)
    assert rc in (xm.XM_ERR_INVALID_ARGUMENT, xm.XM_ERR_UNSUPPORTED) and msg == message
    ws = ctypes.c_size_t()
    assert getattr(xm.load_library(), f"xm_{op}_workspace_size")(
        ctypes.byref(default_attrs(xm, op)), C._array(xm, tensors), len(tensors), ctypes.byref(ws)) == rc


@pytest.mark.parametrize("op", MAKE)
def test_refused_types_and_counts(xm, op):
    m = C.Maker(xm)
    good = MAKE[op](m)
    attrs = default_attrs(xm, op)
    assert C.shape_query(xm, op, attrs, good)[0] == 0
    assert "inputs" in C.shape_query(xm, op, attrs, good[:-1])[1]
    for i in range(len(good)):
        if i == 0 or good[i].shape[0] == 0:
            continue
        bad = list(good)
        bad[i] = xm.XmTensor.from_buffer_copy(good[i])
        bad[i].dtype = F16 if good[i].dtype != F16 else F32
        rc, msg, _ = C.shape_query(xm, op, attrs, bad)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg, i
        bad[i] = xm.XmTensor.from_buffer_copy(good[i])
        bad[i].data = None
        assert "has no data" in C.shape_query(xm, op, attrs, bad)[1]
    lib = xm.load_library()
    assert getattr(lib, f"xm_{op}_output_shape")(None, C._array(xm, good), len(good), None, None) != 0
    assert getattr(lib, f"xm_{op}_output_shape")(ctypes.byref(attrs), None, len(good), None, None) != 0


def test_refused_outputs(xm):
    m = C.Maker(xm)
    refuse = lambda op, attrs, t, outs: C.fwd(xm, op, attrs, t, outs)  # noqa: E731
    t = gate_in(m, init=(2, 8))
    y, s = m((2, 16, 8), BF16), m((2, 8))
    a = attrs_of(xm, "gated_recurrence", 1)
    for outs, message in (
        ([m((2, 16, 8), F16), s], "output must have the shape and type of x"),
        ([y, m((2, 9))], "final_state must have the shape and type of the state input"),
        ([y, m((2, 8), BF16)], "final_state must have the shape and type of the state input"),
        ([y, m((2, 8), F32, t[3].data + 4)], "final_state must not overlap the state input unless it is the same tensor"),
        ([m((2, 16, 8), BF16, t[0].data), s], "an output must not overlap an input"),
        ([m((2, 16, 8), BF16, t[1].data + 16), s], "an output must not overlap an input"),
        ([y, m((2, 8), F32, y.data + 16)], "the outputs must not overlap"),
    ):
        rc, msg = refuse("gated_recurrence", a, t, outs)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg == message
    pool = gate_in(m, init=(5, 8), slots=(2,))
    assert refuse("gated_recurrence", a, pool, [y, m((5, 8))])[1] == \
        "final_state must be the state input itself when state_indices is given"
    u = update_in(m, state=(7, 8), slots=(3,))
    assert refuse("gated_recurrence_update", attrs_of(xm, "gated_recurrence_update"), u, [m((3, 8), BF16), m((7, 8))])[1] == \
        "new_state must be the state input itself when state_indices is given"

    t = grad_in(m, init=(2, 8))
    a = attrs_of(xm, "gated_recurrence_grad", 1, 1)
    dx, df, lb, d0 = m((2, 16, 8), BF16), m((2, 16, 8), BF16), m((8,)), m((2, 8))
    for outs, message in (
        ([m((2, 16, 7), BF16), df, lb, d0], "output must have the shape and type of dy"),
        ([dx, m((2, 16, 8)), lb, d0], "output must have the shape and type of dy"),
        ([dx, df, m((7,)), d0], "d_lower_bound must be float32 with shape (dim)"),
        ([dx, df, m((8,), BF16), d0], "d_lower_bound must be float32 with shape (dim)"),
        ([dx, df, lb, m((3, 8))], "d_initial_state must be float32 with shape (sequences, dim)"),
        ([m((2, 16, 8), BF16, t[0].data), df, lb, d0], "an output must not overlap an input"),
        ([dx, df, lb, m((2, 8), F32, t[5].data)], "an output must not overlap an input"),
        ([dx, m((2, 16, 8), BF16, dx.data), lb, d0], "the outputs must not overlap"),
    ):
        rc, msg = refuse("gated_recurrence_grad", a, t, outs)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg == message

    t = norm_in(m, res=(2, 5, 8))
    a = attrs_of(xm, "layer_norm", 1e-5, 0, 1)
    y, s, st = m((2, 5, 8), BF16), m((2, 5, 8), BF16), m((2, 5, 2))
    for outs, message in (
        ([m((2, 5, 8), F16), s, st], "output must have the shape and type of x"),
        ([y, m((2, 5, 7), BF16), st], "output must have the shape and type of x"),
        ([y, s, m((2, 5, 1))], "stats must be float32 with shape x's with a last axis of 2"),
        ([m((2, 5, 8), BF16, t[0].data), s, st], "an output must not overlap an input"),
        ([m((2, 5, 8), BF16, t[3].data), s, st], "an output must not overlap an input"),
        ([y, m((2, 5, 8), BF16, t[3].data + 2), st], "an output must not overlap an input"),
        ([y, m((2, 5, 8), BF16, t[0].data), st], "an output must not overlap an input"),
        ([y, m((2, 5, 8), BF16, y.data), st], "the outputs must not overlap"),
    ):
        rc, msg = refuse("layer_norm", a, t, outs)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg == message

    t = norm_grad_in(m)
    a = attrs_of(xm, "layer_norm_grad", 0, 1)
    dx, dw, db = m((2, 5, 8), BF16), m((8,)), m((8,))
    for outs, message in (
        ([m((2, 5, 8)), dw, db], "output must have the shape and type of dy"),
        ([dx, m((8,), BF16), db], "d_weight must be float32 with shape (dim)"),
        ([dx, dw, m((9,))], "d_bias must be float32 with shape (dim)"),
        ([dx, dw, m((8,), F32, dw.data)], "the outputs must not overlap"),
        ([m((2, 5, 8), BF16, t[1].data), dw, db], "an output must not overlap an input"),
    ):
        rc, msg = refuse("layer_norm_grad", a, t, outs)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg == message


def test_empty_calls_need_no_device(xm):
    m = C.Maker(xm)
    run = lambda op, attrs, t, outs: C.fwd(xm, op, attrs, t, outs)[0]  # noqa: E731
    assert run("gated_recurrence", attrs_of(xm, "gated_recurrence"), gate_in(m, x=(2, 0, 8)), [m((2, 0, 8), BF16)]) == 0
    t = gate_in(m, x=(0, 4, 8), init=(64, 8))
    assert run("gated_recurrence", attrs_of(xm, "gated_recurrence", 1), t, [m((0, 4, 8), BF16), t[3]]) == 0
    t = update_in(m, x=(0, 8), state=(64, 8))
    assert run("gated_recurrence_update", attrs_of(xm, "gated_recurrence_update"), t, [m((0, 8), BF16), t[3]]) == 0
    assert run("gated_recurrence_grad", attrs_of(xm, "gated_recurrence_grad", 0, 1), grad_in(m, dy=(0, 4, 8)),
               [m((0, 4, 8), BF16), m((0, 4, 8), BF16), m((0, 8))]) == 0
    assert run("layer_norm", attrs_of(xm, "layer_norm"), norm_in(m, x=(0, 8)), [m((0, 8), BF16)]) == 0
    assert run("layer_norm_grad", attrs_of(xm, "layer_norm_grad"), norm_grad_in(m, dy=(0, 8), weight=(0,), stats=(0, 2)),
               [m((0, 8), BF16)]) == 0


def test_python_refuses_host_tensors_and_missing_inputs(xm):
    x, s = torch.zeros(2, 8, 16), torch.zeros(2, 16)
    for call, match in (
        (lambda: xm.GatedRecurrenceFn(x, x), "x must be a CUDA tensor"),
        (lambda: xm.GatedRecurrenceFn(x[0], x[0], output_final_state=1), "x must have rank 3"),
        (lambda: xm.GatedRecurrenceFn(None, None), "x must be a CUDA tensor"),
        (lambda: xm.GatedRecurrenceGradFn(x, x, x, x), "dy must be a CUDA tensor"),
        (lambda: xm.GatedRecurrenceGradFn(x[0], x, x, x), "dy must have rank 3"),
        (lambda: xm.GatedRecurrenceGradFn(None, x, x, x), "dy must have rank 3"),
        (lambda: xm.GatedRecurrenceGradFn(x, x, x, x, out=(None,)), "out must hold 4 outputs"),
        (lambda: xm.GatedRecurrenceUpdateFn(x[0], x[0]), "needs a state"),
        (lambda: xm.GatedRecurrenceUpdateFn(s, s, None, s), "x must be a CUDA tensor"),
        (lambda: xm.LayerNormFn(x), "x must be a CUDA tensor"),
        (lambda: xm.LayerNormFn(torch.zeros(())), "x must have at least one axis"),
        (lambda: xm.LayerNormFn(None), "x must have at least one axis"),
        (lambda: xm.LayerNormGradFn(x, x), "needs the forward call's stats"),
        (lambda: xm.LayerNormGradFn(x, x, None, x), "dy must be a CUDA tensor"),
        (lambda: xm.LayerNormGradFn(x, x, None, x, out=(None,)), "out must hold 3 outputs"),
    ):
        with pytest.raises(xm.XmError, match=match):
            call()


# ------------------------------------------------------------------ the definitions


def _leaf(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_()


def _unrolled(x, f, low, h0, segs):
    """The recurrence as its formula says, one token after the other, with autograd."""
    ys, ends = [None] * x.shape[0], []
    for i, (s, e) in enumerate(segs):
        h = h0[i]
        for t in range(s, e):
            a = low + (1 - low) / (1 + torch.exp(-f[t]))
            h = a * h + (1 - a) * x[t]
            ys[t] = h
        ends.append(h)
    return torch.stack(ys), torch.stack(ends)


@pytest.mark.parametrize("cu", [None, [0, 5, 5, 6, 14]])
def test_recurrence_definition_against_autograd(cu):
    g = torch.Generator().manual_seed(3)
    batch, seqlen, dim = (2, 7, 3) if cu is None else (1, 14, 3)
    segs = [(0, 7), (7, 14)] if cu is None else list(zip(cu, cu[1:]))
    x, f, h0 = _leaf(g, 14, dim), _leaf(g, 14, dim), _leaf(g, len(segs), dim)
    low = (torch.rand(dim, generator=g, dtype=torch.float64) * 0.9).requires_grad_()
    y, last = _unrolled(x, f, low, h0, segs)
    shape = (batch, seqlen, dim)
    detached = [v.detach() for v in (x.reshape(shape), f.reshape(shape), low, h0)]
    got, yb, final, fb = Q.recurrence(*detached, cu=cu)
    assert torch.allclose(got.reshape(-1, dim), y, atol=1e-13) and torch.allclose(final, last, atol=1e-13)
    assert float(yb.max()) < 1e-5 and float(fb.max()) < 1e-5
    dy, dl = torch.randn(14, dim, generator=g, dtype=torch.float64), torch.randn(len(segs), dim, generator=g,
                                                                                 dtype=torch.float64)
    want = torch.autograd.grad((y * dy).sum() + (last * dl).sum(), (x, f, low, h0))
    grads = Q.recurrence_grad(dy.reshape(shape), *detached[:2], y.detach().reshape(shape), detached[2], detached[3], cu, dl)
    for (v, b), w in zip(grads, want):
        assert torch.allclose(v.reshape(w.shape), w, atol=1e-12) and float(b.max()) < 1e-4


def test_recurrence_gradients_against_differences():
    g = torch.Generator().manual_seed(4)
    segs, dim = [(0, 4), (4, 9)], 2
    args = [torch.randn(9, dim, generator=g, dtype=torch.float64), torch.randn(9, dim, generator=g, dtype=torch.float64),
            torch.rand(dim, generator=g, dtype=torch.float64) * 0.8, torch.randn(2, dim, generator=g, dtype=torch.float64)]
    dy = torch.randn(9, dim, generator=g, dtype=torch.float64)
    y, _ = _unrolled(*args, segs)
    shape = (1, 9, dim)
    grads = Q.recurrence_grad(dy.reshape(shape), args[0].reshape(shape), args[1].reshape(shape), y.reshape(shape), args[2],
                              args[3], [0, 4, 9])
    loss = lambda a: float((_unrolled(*a, segs)[0] * dy).sum())  # noqa: E731
    for k, (v, _) in enumerate(grads):
        for i in range(args[k].numel()):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[k].view(-1)[i] += 1e-5
            lo[k].view(-1)[i] -= 1e-5
            # central differences: error h^2 f''' / 6 and rounding 1e-16 / h
            assert abs((loss(hi) - loss(lo)) / 2e-5 - float(v.reshape(-1)[i])) < 1e-8


@pytest.mark.parametrize("rms", [False, True])
def test_norm_definition_against_autograd(rms):
    g = torch.Generator().manual_seed(5)
    x, r, w, b = _leaf(g, 6, 11), _leaf(g, 6, 11), _leaf(g, 11), _leaf(g, 11)
    s = x + r
    if rms:
        y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-3) * w + b
    else:
        y = torch.nn.functional.layer_norm(s, (11,), w, b, 1e-3)
    sd = s.detach()
    (got, yb), _, (stats, _) = Q.norm(sd, w.detach(), b.detach(), None, 1e-3, rms)
    assert torch.allclose(got, y, atol=1e-13) and float(yb.max()) < 1e-4
    dy, ds = torch.randn(6, 11, generator=g, dtype=torch.float64), torch.randn(6, 11, generator=g, dtype=torch.float64)
    want = torch.autograd.grad((y * dy).sum() + (s * ds).sum(), (x, r, w, b))
    (dx, db1), (dw, db2), (dbias, db3) = Q.norm_grad(dy, sd, w.detach(), stats, ds, rms)
    for v, wnt in ((dx, want[0]), (dx, want[1]), (dw, want[2]), (dbias, want[3])):
        assert torch.allclose(v, wnt, atol=1e-12)
    assert max(float(v.max()) for v in (db1, db2, db3)) < 1e-4


def test_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(6)
    args = [torch.randn(2, 5, generator=g, dtype=torch.float64) for _ in range(1)] + [
        torch.randn(5, generator=g, dtype=torch.float64) for _ in range(2)]
    dy = torch.randn(2, 5, generator=g, dtype=torch.float64)
    for rms in (False, True):
        value = lambda a: float((Q.norm(*a, None, 1e-2, rms)[0][0] * dy).sum())  # noqa: E731
        stats = Q.norm(*args, None, 1e-2, rms)[2][0]
        grads = Q.norm_grad(dy, args[0], args[1], stats, None, rms)
        for k, (v, _) in enumerate(grads):
            for i in range(args[k].numel()):
                hi, lo = [a.clone() for a in args], [a.clone() for a in args]
                hi[k].view(-1)[i] += 1e-5
                lo[k].view(-1)[i] -= 1e-5
                assert abs((value(hi) - value(lo)) / 2e-5 - float(v.reshape(-1)[i])) < 1e-7
