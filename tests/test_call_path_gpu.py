"""The Python call path of the serving and layer operators on the GPU: errors that
come from torch, other threads."""

from __future__ import annotations

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
