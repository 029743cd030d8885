"""Edges of the serving operators that need no GPU: what an empty optional input
means, limits, and what the sources promise to the compiler."""

from __future__ import annotations

import torch


def test_empty_indices_allocate_the_state_output(xm):
    """An empty state_indices or cu_seqlens counts as absent, in the Python mirror as in the library."""
    x, state, none = torch.zeros(3, 8, 20), torch.zeros(3, 8, 4), torch.empty(0, dtype=torch.int32)
    row, slots = (8, 4), torch.zeros(3, dtype=torch.int32)
    shape = xm._prompt_state_shape
    for empty in (None, none):
        for cu in (None, none):
            assert shape(x, cu, empty, state, None, row) == (3, 8, 4)
            assert shape(x, cu, empty, None, None, row) == (3, 8, 4)
            assert shape(x, cu, slots, state, None, row) is None
            assert shape(x, cu, empty, state, state, row) is None
        assert shape(x[:1], torch.tensor([0, 4, 20]), empty, None, None, row) == (2, 8, 4)
