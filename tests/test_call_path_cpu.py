"""The Python call path of the serving and layer operators, without a GPU: the
native entry is replaced by a Python function where one is needed."""

from __future__ import annotations

import pathlib
import shutil
import subprocess
import sys
import sysconfig
import threading
import time
import weakref

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]
SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")


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


def _workspace_of(xm, nbytes):
    """A workspace query that answers with nbytes, as the native call path takes it."""
    c = xm.ctypes

    @c.CFUNCTYPE(c.c_int, c.c_void_p, c.c_void_p, c.c_int32, c.POINTER(c.c_size_t))
    def size(attrs, inputs, n, answer):
        answer[0] = nbytes
        return 0

    return size, c.cast(size, c.c_void_p).value


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs an allocation that fails")
def test_torch_errors_come_through_as_torch_raises_them(xm):
    """A workspace that torch cannot allocate: torch's own exception, without a C++ trace in its text."""
    size, entry = _workspace_of(xm, 1000)
    with pytest.raises(RuntimeError, match="NVIDIA driver") as caught:
        xm._load_pycall().call(0, entry, 0, (), b"", (), 0, -1, None, 0)
    assert "Exception raised from" not in str(caught.value) and "frame #" not in str(caught.value)


def test_the_workspace_query_lets_other_threads_run(xm):
    """The interpreter is free from the workspace query on, so that allocations that wait for the device hold nobody up
    (libc's usleep stands in for the query; it sleeps as many microseconds as its first argument says)."""
    entry = xm.ctypes.cast(xm.ctypes.CDLL(None).usleep, xm.ctypes.c_void_p).value
    none = xm.ctypes.cast(xm.ctypes.CDLL(None).getppid, xm.ctypes.c_void_p).value
    ran = []
    other = threading.Thread(target=lambda: (time.sleep(0.05), ran.append(time.monotonic())))
    other.start()
    xm._load_pycall().call(none, entry, 900_000, (), b"", (), 0, -1, None, 0)
    done = time.monotonic()
    other.join()
    assert ran[0] < done - 0.1


# ------------------------------------------------------------------ building and loading


def _make(where, *args):
    return subprocess.run(["make", "-C", str(where), f"PYTHON={sys.executable}", *args], check=True, capture_output=True,
                          text=True).stdout


@pytest.fixture
def built(tmp_path):
    """A copy of the package that counts as built against torch 1.0."""
    pkg = tmp_path / "pkg"
    shutil.copytree(ROOT / "include", tmp_path / "include")
    shutil.copytree(ROOT / "xmetai-onnx-plugins_b200" / "csrc", pkg / "csrc")
    shutil.copy(ROOT / "xmetai-onnx-plugins_b200" / "Makefile", pkg)
    (pkg / "_build").mkdir()
    _make(pkg, "-t", "TORCH_VERSION=1.0")
    return pkg


def test_the_call_path_is_built_anew_for_another_torch(built):
    assert "pycall" not in _make(built, "-n", "TORCH_VERSION=1.0")
    plan = _make(built, "-n", "TORCH_VERSION=2.0")
    assert "pycall.cpp" in plan and "-o libxm_ops.so" not in plan
    # and once more when the first one comes back
    stamp = f"_build/call{SUFFIX}.torch-%s"
    _make(built, "TORCH_VERSION=2.0", stamp % "2.0")
    assert (built / (stamp % "2.0")).exists() and not (built / (stamp % "1.0")).exists()
    assert "pycall.cpp" in _make(built, "-n", "TORCH_VERSION=1.0")


def test_the_c_library_builds_beside_a_torch_without_cuda(built, tmp_path):
    (tmp_path / "torch" / "include" / "ATen").mkdir(parents=True)
    (tmp_path / "torch" / "lib").mkdir()
    plan = _make(built, "-n", "-B", f"TORCH={tmp_path / 'torch'}")
    assert "-o libxm_ops.so" in plan and "pycall.cpp" not in plan


def test_a_call_path_of_another_torch_is_refused(xm, monkeypatch, tmp_path):
    """With how to build it, whether it can be loaded or not."""
    how = f"build it with `make -C .* PYTHON={sys.executable}`"
    monkeypatch.setattr(xm, "_pycall", None)
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "0.0.1")
        with pytest.raises(xm.XmError, match=f"was built for torch .*, this is 0.0.1; {how}"):
            xm._load_pycall()
    monkeypatch.setattr(xm, "_PKG_DIR", tmp_path)
    with pytest.raises(xm.XmError, match=f"not found; {how}"):
        xm._load_pycall()
    # a module that needs what this torch does not have
    (tmp_path / "m.c").write_text("void missing(void); void *PyInit__xm_call(void) { missing(); return 0; }")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / ("_xm_call" + SUFFIX)), str(tmp_path / "m.c")], check=True)
    with pytest.raises(xm.XmError, match=f"cannot be loaded.*missing.*; {how}"):
        xm._load_pycall()
    monkeypatch.undo()
    assert xm._load_pycall() is not None
