"""The Python call path of the serving and layer operators on the GPU: errors that
come from torch, other threads."""

from __future__ import annotations

import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_out_of_memory_is_torchs(xm, cuda):
    """A copy and a workspace that do not fit raise torch.OutOfMemoryError, and the next call works."""
    from test_call_path_cpu import _workspace_of

    wide = torch.zeros(1, 1, 1, device="cuda").expand(1, 2**20, 2**20)  # 4 TB once it is copied
    x = torch.rand(3, 8, device="cuda")
    want = xm.LayerNormFn(x)
    for call in (lambda: xm.GatedRecurrenceFn(wide, wide), lambda: xm.SelectiveScanVarlenFn(
            wide, wide, torch.zeros(2**20, 1, device="cuda"), *[torch.zeros(1, 2**20, 1, device="cuda")] * 2)):
        with pytest.raises(torch.OutOfMemoryError):
            call()
        assert torch.equal(xm.LayerNormFn(x), want)
    size, entry = _workspace_of(xm, 2**42)
    with pytest.raises(torch.OutOfMemoryError):
        xm._load_pycall().call(0, entry, 0, (), b"", (), 0, -1, None, 0)
    assert torch.equal(xm.LayerNormFn(x), want)


def test_too_many_axes(xm, cuda):
    x = torch.rand(1, 1, 1, 1, 1, 1, 1, 2, 8, device="cuda")
    with pytest.raises(ValueError, match="tensor rank above 8 is not supported"):
        xm.LayerNormFn(x)
    with pytest.raises(ValueError, match="tensor rank above 8 is not supported"):
        xm.CausalConv1dUpdateFn(x, x, None, x)
    assert xm.LayerNormFn(x[0]).shape == x.shape[1:]


def test_other_threads_run_during_a_call(xm, cuda):
    """serve() with libc's usleep in place of the workspace query (which sleeps as long as its first argument says)."""
    xm._NORM.load()
    entry, none = (xm.ctypes.cast(f, xm.ctypes.c_void_p).value for f in (xm.ctypes.CDLL(None).usleep,
                                                                       xm.ctypes.CDLL(None).getppid))
    x = torch.rand(3, 8, device="cuda")
    ran = []
    other = threading.Thread(target=lambda: (time.sleep(0.05), ran.append(time.monotonic())))
    other.start()
    xm._load_pycall().serve(none, entry, 900_000, (x, None, None, None), xm._NORM.blanks, (None,), (None,), -1)
    done = time.monotonic()
    other.join()
    assert ran[0] < done - 0.1


def test_calls_from_several_threads(xm, cuda):
    """Threads with a stream each call with attributes, strides and outputs of their own; all get what one thread gets."""
    x = torch.rand(64, 100, device="cuda")
    cases = [(x[:, i:i + 40], 10.0**-i, i % 2) for i in range(6)]

    def run(case):
        v, eps, rms = case
        y, stats = xm.LayerNormFn(v, eps=eps, rms=rms, output_stats=1)
        s = torch.ones(64, 40, device="cuda")
        return y, stats, *xm.GatedRecurrenceUpdateFn(v, y, None, s), xm.GatedRecurrenceFn(v[None], y[None]), \
            xm.LayerNormGradFn(y, v, None, stats, rms=rms, output_bias_grad=1)[2]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(cases))

    def worker(case, expected):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait(30)
            for _ in range(200):
                got = run(case)
            torch.cuda.current_stream().synchronize()
            wrong.extend(k for k, (a, b) in enumerate(zip(got, expected)) if not torch.equal(a, b))

    threads = [threading.Thread(target=worker, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert wrong == [] and not any(t.is_alive() for t in threads)


def test_a_residual_without_rows(xm, cuda):
    """It counts as a residual, and is checked like one, where it has x's shape; any other empty tensor is absent."""
    x, w = torch.empty(0, 24, device="cuda"), torch.rand(24, device="cuda")
    none = torch.empty(0, device="cuda")
    y, s, st = xm.LayerNormFn(x, w, None, x.clone(), output_stats=1)
    assert y.shape == s.shape == x.shape and st.shape == (0, 2)
    kept = torch.empty(0, 24, device="cuda")
    assert xm.LayerNormFn(x, w, None, kept, residual_out=kept)[1] is kept
    # absent: the same results as where x has rows
    assert xm.LayerNormFn(x, w, None, none).shape == x.shape
    y, st = xm.LayerNormFn(x, w, None, none, output_stats=1)
    assert y.shape == x.shape and st.shape == (0, 2)
    rows = torch.rand(2, 24, device="cuda")
    assert torch.equal(xm.LayerNormFn(rows, w, None, none), xm.LayerNormFn(rows, w))
    for residual, into, match in ((x.half(), None, "float32"), (x.cpu(), None, "residual must be a tensor on cuda:0"),
                                  (x.clone(), rows, "shape and type of x"), (x.clone(), x.half(), "shape and type of x"),
                                  (x.clone(), x.cpu(), "an output must be a contiguous tensor on cuda:0")):
        with pytest.raises(xm.XmError, match=match):
            xm.LayerNormFn(x, w, None, residual, residual_out=into)


def _functions(xm):
    """The operators and their gradients in autograd's terms, as a program that uses it wires them."""

    class GatedRecurrence(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, f, lower_bound, h0, cu):
            y, h_last = xm.GatedRecurrenceFn(x, f, lower_bound, h0, cu, output_final_state=1)
            ctx.save_for_backward(x, f, y, lower_bound, h0, cu)
            return y, h_last

        @staticmethod
        def backward(ctx, dy, d_last):
            x, f, y, lower_bound, h0, cu = ctx.saved_tensors
            return (*xm.GatedRecurrenceGradFn(dy, x, f, y, lower_bound, h0, cu, d_last), None)

    class ResidualNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, residual):
            y, s, stats = xm.LayerNormFn(x, weight, bias, residual, output_stats=1)
            ctx.save_for_backward(s, weight, stats)
            return y, s

        @staticmethod
        def backward(ctx, dy, ds):
            s, weight, stats = ctx.saved_tensors
            dx, d_weight, d_bias = xm.LayerNormGradFn(dy, s, weight, stats, ds, output_bias_grad=1)
            return dx, d_weight, d_bias, dx

    return GatedRecurrence.apply, ResidualNorm.apply


def test_in_autograd_functions(xm, cuda):
    """A layer of both in a program that uses autograd: the gradients are those of the formulas, by autograd in 64 bits.
    Every operator is off by about 2^-20 of what it sums, and gates of at most 1 - 0.3 / (1 + e^4) keep some two hundred
    tokens at most: 2^-13 of the largest value."""
    recurrence, norm = _functions(xm)
    g = torch.Generator().manual_seed(81)
    n, dim = 130, 24
    leaves = [torch.randn(1, n, dim, generator=g), 1 + 0.1 * torch.randn(dim, generator=g), torch.randn(dim, generator=g),
              torch.randn(1, n, dim, generator=g), 0.7 * torch.rand(dim, generator=g), torch.randn(2, dim, generator=g)]
    cu, weights = [0, 50, n], torch.randn(n, 1, dim, generator=g)
    dev = [t.cuda().requires_grad_() for t in leaves]
    x, w, b, r, low, h0 = dev
    h, s = norm(x, w, b, r)
    y, last = recurrence(h, s.clamp(-4, 4), low, h0, torch.tensor(cu).cuda())
    # (a transposed gradient: not contiguous)
    loss = (y.transpose(0, 1) * weights.cuda()).sum() + (last * last).sum() + s.sum()
    got = torch.autograd.grad(loss, dev)

    x, w, b, r, low, h0 = exact = [t.double().requires_grad_() for t in leaves]
    s = x + r
    d = s - s.mean(-1, keepdim=True)
    h = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * w + b
    a = low + (1 - low) * torch.sigmoid(s.clamp(-4, 4))
    ys, last = [], []
    for i, (p, q) in enumerate(zip(cu, cu[1:])):
        state = h0[i]
        for t in range(p, q):
            state = a[0, t] * state + (1 - a[0, t]) * h[0, t]
            ys.append(state)
        last.append(state)
    last = torch.stack(last)
    loss = (torch.stack(ys).unsqueeze(1) * weights.double()).sum() + (last * last).sum() + s.sum()
    for k, (u, v) in enumerate(zip(got, torch.autograd.grad(loss, exact))):
        assert float((u.cpu().double() - v).abs().max()) <= 2.0**-13 * float(v.abs().max()), k
