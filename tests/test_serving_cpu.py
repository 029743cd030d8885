"""The serving operators without a GPU: attribute defaults, shape and workspace
queries, what each refuses, and their float64 definitions against independent
ones. Validation never touches tensor memory, so fake device addresses do."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import serving_reference as R

F32, I32, I64, F16, BF16 = 1, 6, 7, 10, 16


class Maker:
    """Descriptors at distinct fake addresses, never dereferenced."""

    def __init__(self, xm):
        self.xm, self.next = xm, 1 << 20

    def __call__(self, shape, dtype=F32, data=None):
        t = self.xm.XmTensor()
        n = int(np.prod(shape, dtype=object)) if len(shape) else 1
        if data is None:
            data, self.next = self.next, self.next + (n * 8 + 4096) // 256 * 256
        t.data = data if n > 0 else None
        for i, s in enumerate(shape):
            t.shape[i] = s
        t.rank, t.dtype = len(shape), dtype
        return t


def _array(xm, tensors):
    a = (xm.XmTensor * len(tensors))()
    for i, t in enumerate(tensors):
        a[i] = t
    return a


def shape_query(xm, op, attrs, tensors):
    lib = xm.load_library()
    shape, rank = (ctypes.c_int64 * 8)(), ctypes.c_int32()
    rc = getattr(lib, f"xm_{op}_output_shape")(ctypes.byref(attrs), _array(xm, tensors), len(tensors), shape,
                                               ctypes.byref(rank))
    return rc, lib.xm_last_error().decode(), tuple(shape[i] for i in range(rank.value))


def fwd(xm, op, attrs, tensors, outs):
    """Calls that are rejected return before any device work."""
    lib = xm.load_library()
    rc = getattr(lib, f"xm_{op}_fwd")(ctypes.byref(attrs), _array(xm, tensors), len(tensors), _array(xm, outs), None, 0,
                                     None)
    return rc, lib.xm_last_error().decode()


def conv_in(m, io=BF16, x=(2, 8, 16), w=(8, 4), bias=(8,), init=(0,), cu=(0,), slots=(0,), live=(0,), cudt=I32):
    return [m(x, io), m(w), m(bias), m(init, io), m(cu, cudt), m(slots, I32), m(live, I64)]


def scan_in(m, io=BF16, u=(2, 16, 8), A=(8, 4), B=(2, 16, 1, 4), C=None, D=(8,), z=(0,), bias=(8,), init=(0,), cu=(0,),
            slots=(0,), live=(0,)):
    return [m(u, io), m(u, io), m(A), m(B, io), m(C or B, io), m(D), m(z, io), m(bias), m(init), m(cu, I32),
            m(slots, I64), m(live, I32)]


def update_in(m, io=BF16, u=(3, 8), A=(8, 4), B=(3, 4), D=(8,), z=(0,), bias=(0,), state=(3, 8, 4), slots=(0,)):
    return [m(u, io), m(u, io), m(A), m(B, io), m(B, io), m(D), m(z, io), m(bias), m(state), m(slots, I32)]


def conv_update_in(m, io=BF16, x=(3, 8), w=(8, 4), bias=(8,), state=(3, 8, 3), slots=(0,)):
    return [m(x, io), m(w), m(bias), m(state, io), m(slots, I32)]


def test_attribute_defaults(xm):
    lib = xm.load_library()
    c, cu, s, su = xm.CausalConv1dAttrs(9, 9, 9), xm.CausalConv1dUpdateAttrs(9), xm.SelectiveScanVarlenAttrs(9, 9), \
        xm.SelectiveStateUpdateAttrs(9)
    lib.xm_causal_conv1d_attrs_default(ctypes.byref(c))
    lib.xm_causal_conv1d_update_attrs_default(ctypes.byref(cu))
    lib.xm_selective_scan_varlen_attrs_default(ctypes.byref(s))
    lib.xm_selective_state_update_attrs_default(ctypes.byref(su))
    assert (c.silu, c.channels_last, c.output_final_state) == (1, 0, 0)
    assert cu.silu == 1 and (s.delta_softplus, s.output_final_state) == (0, 0) and su.delta_softplus == 0
    for op, a in (("causal_conv1d", c), ("causal_conv1d_update", cu), ("selective_scan_varlen", s),
                  ("selective_state_update", su)):
        assert getattr(lib, f"xm_{op}_check_attrs")(ctypes.byref(a)) == 0
        assert getattr(lib, f"xm_{op}_check_attrs")(None) == xm.XM_ERR_INVALID_ARGUMENT
    assert {"CausalConv1dFn", "CausalConv1dUpdateFn", "SelectiveScanVarlenFn", "SelectiveStateUpdateFn"} <= set(xm.OP_NAMES)


def test_valid_shapes(xm):
    m = Maker(xm)
    conv, scan = xm.CausalConv1dAttrs(1, 0, 0), xm.SelectiveScanVarlenAttrs(1, 0)
    for io in (F32, BF16, F16):
        assert shape_query(xm, "causal_conv1d", conv, conv_in(m, io))[::2] == (0, (2, 8, 16))
        assert shape_query(xm, "causal_conv1d", conv, conv_in(m, io, bias=(0,), init=(2, 8, 3)))[0] == 0
        assert shape_query(xm, "selective_scan_varlen", scan, scan_in(m, io))[::2] == (0, (2, 16, 8))
        assert shape_query(xm, "selective_scan_varlen", scan, scan_in(m, io, B=(2, 16, 4), D=(0,), bias=(0,),
                                                                      z=(2, 16, 8), init=(2, 8, 4)))[0] == 0
        assert shape_query(xm, "selective_state_update", xm.SelectiveStateUpdateAttrs(1), update_in(m, io))[2] == (3, 8)
        assert shape_query(xm, "causal_conv1d_update", xm.CausalConv1dUpdateAttrs(1), conv_update_in(m, io))[2] == (3, 8)
    packed = conv_in(m, x=(1, 16, 8), w=(8, 2), cu=(4,), init=(9, 8, 1), slots=(3,), live=(3,))
    assert shape_query(xm, "causal_conv1d", xm.CausalConv1dAttrs(1, 1, 1), packed)[::2] == (0, (1, 16, 8))
    assert shape_query(xm, "causal_conv1d", conv, conv_in(m, x=(0, 8, 16)))[::2] == (0, (0, 8, 16))
    assert shape_query(xm, "causal_conv1d", conv, conv_in(m, x=(2, 8, 0)))[::2] == (0, (2, 8, 0))


REFUSED = [
    ("causal_conv1d", dict(x=(8, 16)), "x must have rank 3"),
    ("causal_conv1d", dict(w=(7, 4)), "weight must have shape (dim, width)"),
    ("causal_conv1d", dict(w=(8, 5)), "causal convolution width must be 2, 3 or 4"),
    ("causal_conv1d", dict(w=(8, 1)), "causal convolution width must be 2, 3 or 4"),
    ("causal_conv1d", dict(bias=(4,)), "bias must be empty or have shape (dim)"),
    ("causal_conv1d", dict(init=(2, 8, 4)), "initial_state must have shape (sequences, dim, width - 1)"),
    ("causal_conv1d", dict(init=(3, 8, 3)), "initial_state must have shape (sequences, dim, width - 1)"),
    ("causal_conv1d", dict(init=(5, 8), slots=(2,)), "initial_state must have shape (slots, dim, width - 1)"),
    ("causal_conv1d", dict(slots=(2,)), "state_indices needs a non-empty initial_state"),
    ("causal_conv1d", dict(init=(5, 8, 3), slots=(3,)), "state_indices must be empty or have one element per sequence"),
    ("causal_conv1d", dict(live=(3,)), "has_initial_state must be empty or have one element per sequence"),
    ("causal_conv1d", dict(cu=(3,)), "CausalConv1dFn with cu_seqlens expects batch 1"),
    ("causal_conv1d", dict(x=(1, 8, 16), cu=(1,)), "cu_seqlens must be 1-D with at least 2 offsets"),
    ("causal_conv1d", dict(x=(1, 8, 16), cu=(3,), cudt=F32), "cu_seqlens must be int64 or int32"),
    ("causal_conv1d", dict(x=(70000, 8, 40000)), "CausalConv1dFn of 2^31 - 4096 tokens or more is not supported"),
    ("causal_conv1d", dict(x=(1, 8, (1 << 31) - 4096)), "CausalConv1dFn of 2^31 - 4096 tokens or more is not supported"),
    ("causal_conv1d", dict(x=(1, (1 << 30) + 1, 2), w=((1 << 30) + 1, 4), bias=(0,)), "dim above 2^30 is not supported"),
    ("selective_state_update", dict(u=(1, (1 << 30) + 1), A=((1 << 30) + 1, 4), B=(1, 4), D=(0,),
                                    state=(1, (1 << 30) + 1, 4)), "dim above 2^30 is not supported"),
    ("causal_conv1d", dict(x=(2, 8, 1 << 31)), "x dimension is out of range"),
    ("causal_conv1d", dict(x=(1 << 30, 1 << 30, 1 << 30)), "x has too many elements"),
    ("causal_conv1d", dict(x=(2, 8, -1)), "x has a negative dimension"),
    ("selective_scan_varlen", dict(u=(16, 8)), "u must have rank 3"),
    ("selective_scan_varlen", dict(A=(7, 4)), "A must have shape (dim, d_state)"),
    ("selective_scan_varlen", dict(A=(8, 257), B=(2, 16, 1, 257)), "d_state must be 1 to 256"),
    ("selective_scan_varlen", dict(A=(8, 0), B=(2, 16, 1, 0)), "d_state must be 1 to 256"),
    ("selective_scan_varlen", dict(B=(2, 15, 1, 4)), "B must have shape (batch, seqlen, n_groups, d_state)"),
    ("selective_scan_varlen", dict(B=(2, 16, 1, 5)), "B must have shape (batch, seqlen, n_groups, d_state)"),
    ("selective_scan_varlen", dict(C=(2, 16, 2, 4)), "C shape must match B"),
    ("selective_scan_varlen", dict(B=(2, 16, 3, 4)), "dim must be divisible by n_groups"),
    ("selective_scan_varlen", dict(z=(2, 16, 9)), "z shape must match u"),
    ("selective_scan_varlen", dict(D=(9,)), "D must be empty or have shape (dim)"),
    ("selective_scan_varlen", dict(bias=(9,)), "delta_bias must be empty or have shape (dim)"),
    ("selective_scan_varlen", dict(init=(2, 8, 5)), "initial_state must have shape (sequences, dim, d_state)"),
    ("selective_scan_varlen", dict(cu=(3,)), "SelectiveScanVarlenFn with cu_seqlens expects batch 1"),
    ("selective_state_update", dict(state=(2, 8, 4)), "state must have shape (sequences, dim, d_state)"),
    ("selective_state_update", dict(state=(0,)), "SelectiveStateUpdateFn needs a non-empty state"),
    ("selective_state_update", dict(B=(3, 3, 4)), "dim must be divisible by n_groups"),
    ("selective_state_update", dict(B=(2, 4)), "B must have shape (batch, n_groups, d_state)"),
    ("causal_conv1d_update", dict(state=(3, 8, 4)), "state must have shape (sequences, dim, width - 1)"),
    ("causal_conv1d_update", dict(state=(0,)), "CausalConv1dUpdateFn needs a non-empty state"),
    ("causal_conv1d_update", dict(x=(3, 8, 1)), "x must have rank 2"),
]
MAKE = dict(causal_conv1d=conv_in, selective_scan_varlen=scan_in, selective_state_update=update_in,
            causal_conv1d_update=conv_update_in)


def _attrs(xm, op, state=0):
    return dict(causal_conv1d=xm.CausalConv1dAttrs(1, 0, state), causal_conv1d_update=xm.CausalConv1dUpdateAttrs(1),
                selective_scan_varlen=xm.SelectiveScanVarlenAttrs(1, state),
                selective_state_update=xm.SelectiveStateUpdateAttrs(1))[op]


@pytest.mark.parametrize("op,change,message", REFUSED)
def test_refused_inputs(xm, op, change, message):
    tensors = MAKE[op](Maker(xm), **change)
    rc, msg, _ = shape_query(xm, op, _attrs(xm, op), tensors)
    assert rc in (xm.XM_ERR_INVALID_ARGUMENT, xm.XM_ERR_UNSUPPORTED) and msg == message
    ws = ctypes.c_size_t()
    assert getattr(xm.load_library(), f"xm_{op}_workspace_size")(
        ctypes.byref(_attrs(xm, op)), _array(xm, tensors), len(tensors), ctypes.byref(ws)) == rc


@pytest.mark.parametrize("op", MAKE)
def test_refused_types_and_counts(xm, op):
    m = Maker(xm)
    good = MAKE[op](m)
    attrs = _attrs(xm, op)
    assert shape_query(xm, op, attrs, good)[0] == 0
    assert "inputs" in shape_query(xm, op, attrs, good[:-1])[1]
    for i in range(len(good)):
        if i == 0 or good[i].shape[0] == 0:
            continue
        bad = list(good)
        bad[i] = xm.XmTensor.from_buffer_copy(good[i])
        bad[i].dtype = F16 if good[i].dtype != F16 else F32
        rc, msg, _ = shape_query(xm, op, attrs, bad)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg, i
        bad[i] = xm.XmTensor.from_buffer_copy(good[i])
        bad[i].data = None
        assert "has no data" in shape_query(xm, op, attrs, bad)[1]
    lib = xm.load_library()
    assert getattr(lib, f"xm_{op}_output_shape")(None, _array(xm, good), len(good), None, None) != 0
    assert getattr(lib, f"xm_{op}_output_shape")(ctypes.byref(attrs), None, len(good), None, None) != 0


def test_refused_outputs(xm):
    m = Maker(xm)
    a = xm.CausalConv1dAttrs(1, 0, 1)
    t = conv_in(m, init=(2, 8, 3))
    y, s = m((2, 8, 16), BF16), m((2, 8, 3), BF16)
    for outs, message in (
        ([m((2, 8, 15), BF16), s], "output must have the shape and type of x"),
        ([m((2, 8, 16), F16), s], "output must have the shape and type of x"),
        ([y, m((2, 8, 4), BF16)], "final_state must have the shape and type of the state input"),
        ([y, m((2, 8, 3), F32)], "final_state must have the shape and type of the state input"),
        ([m((2, 8, 16), BF16, t[0].data), s], "an output must not overlap an input"),
        ([m((2, 8, 16), BF16, t[0].data + 32), s], "an output must not overlap an input"),
        ([y, m((2, 8, 3), BF16, t[3].data + 2)], "final_state must not overlap the state input unless it is the same tensor"),
        ([y, m((2, 8, 3), BF16, y.data + 64)], "the outputs must not overlap"),
        ([y, m((2, 8, 3), BF16, t[1].data)], "an output must not overlap an input"),
    ):
        rc, msg = fwd(xm, "causal_conv1d", a, t, outs)
        assert rc == xm.XM_ERR_INVALID_ARGUMENT and msg == message
    pool = conv_in(m, init=(5, 8, 3), slots=(2,))
    rc, msg = fwd(xm, "causal_conv1d", a, pool, [y, m((5, 8, 3), BF16)])
    assert msg == "final_state must be the state input itself when state_indices is given"
    rc, msg = fwd(xm, "causal_conv1d", a, pool, [y, m((2, 8, 3), BF16)])
    assert msg == "final_state must have the shape and type of the state input"
    u = update_in(m, state=(7, 8, 4), slots=(3,))
    rc, msg = fwd(xm, "selective_state_update", xm.SelectiveStateUpdateAttrs(1), u, [m((3, 8), BF16), m((7, 8, 4))])
    assert msg == "new_state must be the state input itself when state_indices is given"
    u = update_in(m)
    rc, msg = fwd(xm, "selective_state_update", xm.SelectiveStateUpdateAttrs(1), u, [m((3, 8), BF16, u[8].data), u[8]])
    assert msg == "an output must not overlap an input"
    c = conv_update_in(m)
    rc, msg = fwd(xm, "causal_conv1d_update", xm.CausalConv1dUpdateAttrs(1), c, [m((3, 8), BF16, c[0].data), c[3]])
    assert msg == "an output must not overlap an input"


def test_empty_calls_need_no_device(xm):
    m = Maker(xm)
    assert fwd(xm, "causal_conv1d", xm.CausalConv1dAttrs(1, 0, 0), conv_in(m, x=(2, 8, 0)), [m((2, 8, 0), BF16)])[0] == 0
    assert fwd(xm, "selective_scan_varlen", xm.SelectiveScanVarlenAttrs(1, 0), scan_in(m, u=(0, 16, 8), B=(0, 16, 1, 4)),
               [m((0, 16, 8), BF16)])[0] == 0
    assert fwd(xm, "selective_state_update", xm.SelectiveStateUpdateAttrs(1),
               update_in(m, u=(0, 8), B=(0, 4), state=(0, 8, 4)), [m((0, 8), BF16), m((0, 8, 4))])[0] == 0
    assert fwd(xm, "causal_conv1d_update", xm.CausalConv1dUpdateAttrs(1), conv_update_in(m, x=(0, 8), state=(0, 8, 3)),
               [m((0, 8), BF16), m((0, 8, 3), BF16)])[0] == 0


def test_python_refuses_host_tensors_and_missing_states(xm):
    x, w = torch.zeros(2, 8, 16), torch.zeros(8, 4)
    with pytest.raises(xm.XmError, match="x must be a CUDA tensor"):
        xm.CausalConv1dFn(x, w)
    with pytest.raises(xm.XmError, match="x must have rank 3"):
        xm.CausalConv1dFn(x[0], w, output_final_state=1)
    with pytest.raises(xm.XmError, match="u must be a CUDA tensor"):
        xm.SelectiveScanVarlenFn(x, x, w, x, x)
    with pytest.raises(xm.XmError, match="needs a state"):
        xm.CausalConv1dUpdateFn(x[:, :, 0], w)
    with pytest.raises(xm.XmError, match="needs a state"):
        xm.SelectiveStateUpdateFn(x[:, :, 0], x[:, :, 0], w, x, x)
    with pytest.raises(xm.XmError, match="u must be a CUDA tensor"):
        xm.SelectiveStateUpdateFn(None, None, None, None, None, state=x)


# ------------------------------------------------------------------ the definitions


def test_conv_definition_against_torch():
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(2, 6, 50, generator=g), torch.randn(6, 4, generator=g), torch.randn(6, generator=g)
    y, _, final = R.conv(x, w, b)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.double(), (3, 0)), w.double().unsqueeze(1), b.double(),
                                      groups=6)
    assert torch.allclose(y, torch.nn.functional.silu(want), atol=1e-12)
    assert torch.equal(final, x[:, :, -3:])
    last, _, _ = R.conv(x.transpose(1, 2), w, b, channels_last=True)
    assert torch.equal(last.transpose(1, 2), y)
    # cut at 1 and 20: the states carry
    outs, state = [], None
    for a, c in ((0, 1), (1, 20), (20, 50)):
        p, _, state = R.conv(x[:, :, a:c], w, b, state)
        outs.append(p)
    assert torch.equal(torch.cat(outs, 2), y) and torch.equal(state, final)


def test_scan_definition_against_the_oracle():
    import oracle
    from xmetai_onnx_plugins_b200 import workloads as W

    x = W.ss_inputs(seed=4, batch=2, dim=12, seqlen=40, dstate=16, groups=2)
    want, last = oracle.ss(*[x[k] for k in W.SS_ORDER], softplus=True, gate=True), None
    t = lambda k: torch.from_numpy(x[k]).transpose(1, 2).contiguous()  # noqa: E731
    bc = lambda k: torch.from_numpy(x[k]).permute(0, 3, 1, 2).contiguous()  # noqa: E731
    n = lambda k: torch.from_numpy(x[k])  # noqa: E731
    y, bound, _, _ = R.scan(t("u"), t("delta"), n("A"), bc("B"), bc("C"), n("D"), t("z"), n("delta_bias"))
    assert np.abs(y.transpose(1, 2).numpy() - want).max() <= 1e-10 * np.abs(want).max() and last is None
    assert float(bound.max()) < 1e-3 * float(y.abs().max())


def test_scan_definition_packs_and_continues():
    g = torch.Generator().manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    A, D, bias = -torch.rand(6, 3, generator=g) - 0.1, mk(6), mk(6)
    parts = [(mk(1, n, 6), mk(1, n, 6), mk(1, n, 3), mk(1, n, 3)) for n in (4, 0, 9)]
    pool = mk(5, 6, 3)
    whole = [torch.cat(v, 1) for v in zip(*parts)]
    y, _, final, _ = R.scan(whole[0], whole[1], A, whole[2], whole[3], D, None, bias, state=pool, cu=[0, 4, 4, 13],
                            slots=[3, 0, 9], live=[1, 1, 1])
    for i, (a, c, start) in enumerate(((0, 4, pool[3]), (4, 13, torch.zeros(6, 3)))):
        u, d, B, C = parts[0 if i == 0 else 2]
        one, _, last, _ = R.scan(u, d, A, B, C, D, None, bias, state=start.unsqueeze(0))
        # (float64 exp and log may differ in the last place between vector and scalar code)
        assert torch.allclose(one, y[:, a:c], rtol=1e-12, atol=1e-12)
        if i == 0:
            assert torch.allclose(last[0], final[3], rtol=1e-12, atol=1e-12)
    assert torch.equal(final[[0, 1, 2, 4]], pool[[0, 1, 2, 4]].double())
