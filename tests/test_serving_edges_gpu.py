"""Calls of the serving operators at the edges of what their documentation
allows, on the GPU, against the float64 definitions of serving_reference.py."""

from __future__ import annotations

import pytest
import torch

import serving_reference as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def close(got, want, bound):
    e = R.excess(got, want, bound)
    assert e <= 0, f"off by {e} more than the bound"


# ------------------------------------------------------------------ CausalConv1dFn, addresses


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("batch,seqlen,cu", [(2, 50, None), (1, 9, None), (3, 5, None), (1, 2500, None),
                                             (1, 300, [0, 3, 4, 40, 290]), (1, 40, [6, 9, 33, 40])])
def test_conv_input_and_output_equally_misaligned(xm, cuda, dt, width, batch, seqlen, cu):
    """Channel-major x and out at the same offset from a 16-byte boundary: the first word is cut by x's begin."""
    g = gen(seqlen + width)
    dim = 3
    x, w, b = normal(g, batch, dim, seqlen, dtype=DT[dt]), normal(g, dim, width), normal(g, dim)
    state = normal(g, batch if cu is None else len(cu) - 1, dim, width - 1, dtype=DT[dt])
    before = torch.full_like(x, 5.0)
    y, bound, final = R.conv(x, w, b, state, cu, out=before)
    cud = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    for o in range(1, 16 // x.element_size()):
        src = torch.full((x.numel() + 32,), float("nan"), dtype=x.dtype, device="cuda")
        dst = torch.full((x.numel() + 32,), 5.0, dtype=x.dtype, device="cuda")
        xs, ys = src[o:o + x.numel()].view(x.shape), dst[o:o + x.numel()].view(x.shape)
        xs.copy_(x)
        _, last = xm.CausalConv1dFn(xs, w.cuda(), b.cuda(), state.cuda(), cud, output_final_state=1, out=ys)
        close(ys, y, bound)
        assert torch.equal(last.cpu(), final)
        assert bool((dst[:o] == 5).all()) and bool((dst[o + x.numel():] == 5).all())


# ------------------------------------------------------------------ empty index tensors


def test_empty_index_tensors_are_absent(xm, cuda):
    """Empty state_indices, cu_seqlens and has_initial_state are absent inputs: the given states stay as they were."""
    g = gen(71)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    x, w = normal(g, 2, 20, 8).cuda(), normal(g, 8, 4).cuda()
    state = normal(g, 2, 8, 3).cuda()
    kept = state.clone()
    want = xm.CausalConv1dFn(x, w, None, state, channels_last=1, output_final_state=1)
    got = xm.CausalConv1dFn(x, w, None, state, none, none, none, channels_last=1, output_final_state=1)
    assert got[1] is not state and torch.equal(state, kept)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = xm.CausalConv1dFn(x, w, None, None, none, none, none, channels_last=1, output_final_state=1)
    want = xm.CausalConv1dFn(x, w, channels_last=1, output_final_state=1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    A, B, C = -torch.rand(8, 4).cuda(), normal(g, 2, 20, 4).cuda(), normal(g, 2, 20, 4).cuda()
    state = normal(g, 2, 8, 4).cuda()
    kept = state.clone()
    want = xm.SelectiveScanVarlenFn(x, x, A, B, C, None, None, None, state, delta_softplus=1, output_final_state=1)
    got = xm.SelectiveScanVarlenFn(x, x, A, B, C, None, None, None, state, none, none, none, delta_softplus=1,
                                   output_final_state=1)
    assert got[1] is not state and torch.equal(state, kept)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batch_over_a_pool(xm, cuda):
    """A step without sequences: empty outputs, the pool returned as it was."""
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    w, A = torch.rand(8, 4, device="cuda"), -torch.rand(8, 4, device="cuda")
    cs, ss = torch.rand(5, 8, 3, device="cuda"), torch.rand(5, 8, 4, device="cuda")
    kc, ks = cs.clone(), ss.clone()
    x2, b2 = torch.empty(0, 8, device="cuda"), torch.empty(0, 4, device="cuda")
    x3, b3 = torch.empty(0, 6, 8, device="cuda"), torch.empty(0, 6, 4, device="cuda")
    y, s = xm.CausalConv1dUpdateFn(x2, w, None, cs, none)
    assert y.shape == x2.shape and s is cs
    y, s = xm.SelectiveStateUpdateFn(x2, x2, A, b2, b2, state=ss, state_indices=none)
    assert y.shape == x2.shape and s is ss
    y, s = xm.CausalConv1dFn(x3, w, None, cs, None, none, none, channels_last=1, output_final_state=1)
    assert y.shape == x3.shape and s is cs
    y, s = xm.SelectiveScanVarlenFn(x3, x3, A, b3, b3, None, None, None, ss, None, none, none, output_final_state=1)
    assert y.shape == x3.shape and s is ss
    y, s = xm.SelectiveScanVarlenFn(x3, x3, A, b3, b3, output_final_state=1)
    assert y.shape == x3.shape and s.shape == (0, 8, 4)
    assert torch.equal(cs, kc) and torch.equal(ss, ks)


# ------------------------------------------------------------------ counts near 2^31


def test_single_tokens_of_as_many_sequences_as_allowed(xm, cuda):
    """2^31 - 4097 sequences of one channel, all but a few without a slot: those few are updated once, the others'
    outputs stay as they were. (The counters step past 2^31 behind the last sequence.)"""
    n = 2**31 - 4097
    at = [0, 5, 2**30 + 1, n - 262141, n - 65536, n - 3, n - 1]
    k = len(at)
    pos = torch.tensor(at, device="cuda")
    slots = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    slots[pos] = torch.arange(k, dtype=torch.int32, device="cuda")
    g = gen(91)
    tok = normal(g, k, 1, 1, dtype=torch.bfloat16)
    x = torch.full((n, 1), float("nan"), dtype=torch.bfloat16, device="cuda")
    x[pos] = tok[:, 0].cuda()
    out = torch.full((n, 1), 7.0, dtype=torch.bfloat16, device="cuda")

    def untouched():
        changed = sum(int((part != 7).sum()) for part in out.split(2**28))
        return changed == int((out[pos] != 7).sum())

    w, state = normal(g, 1, 4), normal(g, k, 1, 3, dtype=torch.bfloat16)
    y, bound, final = R.conv(tok, w, None, state, channels_last=True)
    pool = state.cuda()
    xm.CausalConv1dUpdateFn(x, w.cuda(), None, pool, slots, out=out)
    close(out[pos].unsqueeze(1), y, bound)
    assert torch.equal(pool.cpu(), final) and untouched()
    out.fill_(7.0)
    A, D, state = -torch.rand(1, 1, generator=g), normal(g, 1), normal(g, k, 1, 1)
    y, bound, final, ferr = R.scan(tok, tok, A, tok, tok, D, None, None, state)
    pool = state.cuda()
    xm.SelectiveStateUpdateFn(x, x, A.cuda(), x, x, D.cuda(), None, None, pool, slots, delta_softplus=1, out=out)
    close(out[pos].unsqueeze(1), y, bound)
    close(pool, final, ferr)
    assert untouched()


@pytest.mark.parametrize("channels_last", [0, 1])
def test_more_packed_sequences_than_30_bits(xm, cuda, channels_last):
    """2^30 + 4097 sequences of one token, each starting from zeros: y = w_last x, rounded once."""
    n = 2**30 + 4097
    gcuda = torch.Generator(device="cuda").manual_seed(92)
    x = torch.empty(1, n, dtype=torch.bfloat16, device="cuda")
    for part in x[0].split(2**28):
        part.normal_(generator=gcuda)
    w = torch.tensor([[0.7, -1.3]], device="cuda")
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    shape = (1, n, 1) if channels_last else (1, 1, n)
    y = xm.CausalConv1dFn(x.view(shape), w, None, None, cu, silu=0, channels_last=channels_last)
    for a, b in zip(y.view(-1).split(2**28), x.view(-1).split(2**28)):
        assert torch.equal(a, (b.float() * w[0, 1]).to(torch.bfloat16))


# ------------------------------------------------------------------ the scan's join over blocks


SCAN = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


def _run_scan(xm, x, state):
    return xm.SelectiveScanVarlenFn(*[None if x[k] is None else x[k].cuda() for k in SCAN], state.cuda(),
                                    output_final_state=1)


@pytest.mark.parametrize("N", [5, 16])
def test_scan_steps_whose_sum_overflows(xm, cuda, N):
    """Steps of 3e38 over a split axis: each block's sum passes float32's range. The states decay to zero, those with
    A = 0 keep their value, and nothing turns into NaN."""
    g = gen(81)
    tokens, dim = 4096, 6
    x = dict(u=normal(g, 1, tokens, dim), delta=torch.rand(1, tokens, dim, generator=g) * 0.1,
             A=-torch.rand(dim, N, generator=g) - 0.1, B=normal(g, 1, tokens, N), C=normal(g, 1, tokens, N),
             D=None, z=None, delta_bias=None)
    x["A"][:, 0] = 0.0
    huge = slice(500, 2500)
    x["delta"][:, huge] = 3e38
    x["u"][:, huge] = 0.0
    state = normal(g, 1, dim, N)
    y, bound, final, ferr = R.scan(**x, state=state, softplus=False)
    assert torch.isfinite(y).all() and torch.isfinite(final).all()
    got, last = _run_scan(xm, x, state)
    close(got, y, bound)
    close(last, final, ferr)


def test_scan_growth_past_float_range_in_a_block(xm, cuda):
    """Growing states whose factor over a block is above 2^128: zero states stay zero, tiny ones grow to the value that
    token by token gives."""
    g = gen(82)
    tokens, dim, N = 4096, 24, 3
    x = dict(u=torch.zeros(1, tokens, dim), delta=torch.zeros(1, tokens, dim), A=torch.ones(dim, N),
             B=normal(g, 1, tokens, N), C=normal(g, 1, tokens, N), D=None, z=None, delta_bias=None)
    for c in range(dim):
        x["delta"][:, 1000 + 8 * c:1050 + 8 * c, c] = 2.2
    state = torch.zeros(1, dim, N)
    state[:, :, 1] = 1e-30
    state[:, :, 2] = -1e-35
    y, bound, final, ferr = R.scan(**x, state=state, softplus=False)
    assert torch.isfinite(y).all() and float(final.abs().max()) > 1e17
    got, last = _run_scan(xm, x, state)
    close(got, y, bound)
    close(last, final, ferr)


# ------------------------------------------------------------------ streams


def test_streams_of_other_devices_are_refused(xm, cuda):
    """Also the default stream of another device, whose handle equals this one's (a stand-in, so that one GPU does)."""
    from types import SimpleNamespace

    x, w = torch.rand(1, 8, 20, device="cuda"), torch.rand(8, 4, device="cuda")
    here = torch.cuda.default_stream(0)
    assert torch.equal(xm.CausalConv1dFn(x, w, stream=here), xm.CausalConv1dFn(x, w))
    for handle in (here.cuda_stream, torch.cuda.Stream().cuda_stream):
        with pytest.raises(xm.XmError, match="stream belongs to another device"):
            xm.CausalConv1dFn(x, w, stream=SimpleNamespace(device_index=1, cuda_stream=handle))


# ------------------------------------------------------------------ CausalConv1dFn, long rows


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("seqlen,cu", [(1024, None), (2048, None), (2049, None), (8192, None), (8196, None), (16384, None),
                                       (16400, None), (20000, [0, 20000]), (40000, [0, 17000, 17003, 40000])])
def test_conv_rows_around_the_choice_of_runs(xm, cuda, dt, seqlen, cu):
    """Channel-major rows of whole items, of many, and in between, and packed ones, with states."""
    g = gen(seqlen)
    batch = 2 if cu is None else 1
    x, w, b = normal(g, batch, 3, seqlen, dtype=DT[dt]), normal(g, 3, 4), normal(g, 3)
    state = normal(g, batch if cu is None else len(cu) - 1, 3, 3, dtype=DT[dt])
    y, bound, final = R.conv(x, w, b, state, cu)
    got, last = xm.CausalConv1dFn(x.cuda(), w.cuda(), b.cuda(), state.cuda(), None if cu is None else
                                  torch.tensor(cu).cuda(), output_final_state=1)
    close(got, y, bound)
    assert torch.equal(last.cpu(), final)
