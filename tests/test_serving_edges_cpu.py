"""Edges of the serving operators that need no GPU: what an empty optional input
means, limits, and what the sources promise to the compiler."""

from __future__ import annotations

import ctypes
import subprocess
import sys
import sysconfig
import threading
import time

import test_serving_cpu as C
import torch

from conftest import ROOT


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


# ------------------------------------------------------------------ calls without sequences


def test_no_sequences_over_a_pool(xm):
    """Batch 0 with empty state_indices takes a pool of any size and needs no device."""
    m = C.Maker(xm)
    calls = [
        ("causal_conv1d", xm.CausalConv1dAttrs(1, 0, 1), C.conv_in(m, x=(0, 8, 16), init=(64, 8, 3)), 3, (0, 8, 16)),
        ("causal_conv1d", xm.CausalConv1dAttrs(1, 1, 1), C.conv_in(m, x=(0, 16, 8), init=(64, 8, 3)), 3, (0, 16, 8)),
        ("selective_scan_varlen", xm.SelectiveScanVarlenAttrs(1, 1),
         C.scan_in(m, u=(0, 16, 8), B=(0, 16, 1, 4), init=(64, 8, 4)), 8, (0, 16, 8)),
        ("causal_conv1d_update", xm.CausalConv1dUpdateAttrs(1), C.conv_update_in(m, x=(0, 8), state=(64, 8, 3)), 3, (0, 8)),
        ("selective_state_update", xm.SelectiveStateUpdateAttrs(1),
         C.update_in(m, u=(0, 8), B=(0, 4), state=(64, 8, 4)), 8, (0, 8)),
    ]
    for op, attrs, tensors, state, shape in calls:
        assert C.shape_query(xm, op, attrs, tensors)[::2] == (0, shape)
        assert C.fwd(xm, op, attrs, tensors, [m(shape, C.BF16), tensors[state]])[0] == 0
        wrong = list(tensors)
        wrong[state] = m((64, 8, 5), tensors[state].dtype)
        assert "must have shape (sequences, dim" in C.shape_query(xm, op, attrs, wrong)[1]
    state, none = torch.zeros(64, 8, 4), torch.empty(0, dtype=torch.int32)
    assert xm._prompt_state_shape(torch.zeros(0, 6, 8), None, none, state, None, (8, 4)) is None
    assert xm._prompt_state_shape(torch.zeros(0, 6, 8), None, none, None, None, (8, 4)) == (0, 8, 4)


# ------------------------------------------------------------------ what the sources promise


def test_asynchronous_copies_declare_that_they_touch_memory():
    """Plain loads behind a wait, and stores before a copy, are ordered only where the asm statement says so."""
    import re

    statements = []
    for path in sorted((ROOT / "xmetai-onnx-plugins_b200" / "csrc").glob("*.cu*")):
        for m in re.finditer(r'asm volatile\("cp\.async(.*?)\);', path.read_text(), re.S):
            statements.append((path.name, m.group(1)))
    assert len(statements) >= 9
    assert [s for s in statements if '"memory"' not in s[1]] == []


# ------------------------------------------------------------------ limits


def test_scan_refuses_more_channel_blocks_than_a_grid_holds(xm):
    """2^31 blocks of channels are refused by every entry, one sequence less is not."""
    attrs = xm.SelectiveScanVarlenAttrs(1, 0)
    for n, message in ((2**30, "SelectiveScanVarlenFn of 2^31 or more blocks of channels is not supported"),
                       (2**30 - 1, None)):
        m = C.Maker(xm)
        tensors = C.scan_in(m, u=(n, 1, 2), A=(2, 1), B=(n, 1, 2, 1), D=(2,), bias=(0,))
        rc, msg, shape = C.shape_query(xm, "selective_scan_varlen", attrs, tensors)
        ws = ctypes.c_size_t(7)
        size_rc = xm.load_library().xm_selective_scan_varlen_workspace_size(
            ctypes.byref(attrs), C._array(xm, tensors), len(tensors), ctypes.byref(ws))
        if message is None:
            assert (rc, shape, size_rc, ws.value) == (0, (n, 1, 2), 0, 0)
        else:
            assert rc == size_rc == xm.XM_ERR_UNSUPPORTED and msg == message
            rc, msg = C.fwd(xm, "selective_scan_varlen", attrs, tensors, [m((n, 1, 2), C.BF16)])
            assert rc == xm.XM_ERR_UNSUPPORTED and msg == message


# ------------------------------------------------------------------ building


def _make_plan(*args):
    return subprocess.run(["make", "-n", "-B", "-C", str(ROOT / "xmetai-onnx-plugins_b200"), *args], check=True,
                          capture_output=True, text=True).stdout


def test_the_c_library_builds_without_python_headers():
    """`make` leaves the Python call path out where there are no headers for it, and names it by its Python."""
    alone = _make_plan("PYTHON=false")
    assert "-o libxm_ops.so" in alone and "pycall.c" not in alone
    assert "_xm_call" + sysconfig.get_config_var("EXT_SUFFIX") in _make_plan(f"PYTHON={sys.executable}")


def test_build_makes_the_call_path_for_this_python(monkeypatch):
    import __graft_entry__ as entry

    made = []
    monkeypatch.setattr(entry.subprocess, "run", lambda args, **kw: made.append(args))
    entry.build()
    assert f"PYTHON={sys.executable}" in made[0]


def test_the_call_path_lets_other_threads_run(xm):
    """While an operator's entry point runs, the interpreter is free (libc's usleep stands in for one)."""
    entry = ctypes.cast(ctypes.CDLL(None).usleep, ctypes.c_void_p).value
    ran = []
    other = threading.Thread(target=lambda: (time.sleep(0.05), ran.append(time.monotonic())))
    other.start()
    assert xm._load_pycall().call(entry, 0, 900_000, (), b"", (), 0, -1, None, 0) == (0, 0)
    done = time.monotonic()
    other.join()
    assert ran[0] < done - 0.1
