"""The Python call path of the serving and layer operators, without a GPU: the
native entry is replaced by a Python function where one is needed."""

from __future__ import annotations

import threading
import weakref

import pytest
import torch


@pytest.fixture
def native(xm, monkeypatch):
    """Replaces the native entry of LayerNormFn and CausalConv1dUpdateFn: native(f) makes f(attrs' address) run in a call."""

    def install(f):
        for op in (xm._NORM, xm._CONV_UPDATE):
            for name, value in (("fwd", 0), ("size", 0), ("blanks", ()), (
                    "call", lambda fwd, size, attrs, tensors, *rest: (f(attrs), tensors[0], None)[1:])):
                monkeypatch.setattr(op, name, value, raising=False)

    return install


@pytest.mark.parametrize("op", ["norm", "conv"])
def test_attributes_live_as_long_as_the_call(xm, monkeypatch, native, op):
    """Two threads that make the same call at once, held where each has made its struct: it is there, with its values,
    until the call returns."""
    kind = xm.LayerNormAttrs if op == "norm" else xm.CausalConv1dUpdateAttrs
    both, alive = threading.Barrier(2), {}

    class Held(kind):
        def __init__(self, *values):
            super().__init__(*values)
            alive[xm.ctypes.addressof(self)] = weakref.ref(self)
            both.wait(10)

    seen = []

    def entry(address):
        both.wait(10)  # both threads are past making theirs
        struct = alive[address]()
        seen.append(None if struct is None else (struct.eps if op == "norm" else struct.silu))
        both.wait(10)

    native(entry)
    monkeypatch.setattr(xm, kind.__name__, Held)
    x = torch.zeros(2, 4)
    call = (lambda: xm.LayerNormFn(x, eps=0.125)) if op == "norm" else (lambda: xm.CausalConv1dUpdateFn(x, x, None, x))
    threads = [threading.Thread(target=call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert seen == ([0.125] * 2 if op == "norm" else [1] * 2)
