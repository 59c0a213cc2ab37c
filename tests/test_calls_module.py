"""The native module for repeated calls (onnx-rs_b200/_calls.so) is optional: the
package imports without it, beside a file that does not fit, and does not load it
before an operator of the 8-bit linear path is called.  The make rule builds it
anew for another Python or torch."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "onnx-rs_b200")


def run_python(code, where):
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=str(where))
    assert r.returncode == 0, r.stderr[-3000:]
    return r


@pytest.fixture
def package(tmp_path):
    """A copy of the package (links) whose _calls.so can be exchanged."""
    pkg = tmp_path / "onnx-rs_b200"
    pkg.mkdir()
    for name in os.listdir(PKG):
        if name not in ("_calls.so", "__pycache__", "_build", "csrc"):
            os.symlink(os.path.join(PKG, name), pkg / name)
    return pkg


LOAD = """
import importlib, warnings
ob = importlib.import_module("onnx-rs_b200")
assert "_calls.so" not in open("/proc/self/maps").read()
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    print(ob.ops._calls, len(seen), *(w.message for w in seen))
    assert ob.ops._native() is ob.ops._calls and len(seen) <= 1
assert ob.OperatorRegistry.initialize_standard_operators().get_operator("Conv", "", 11) is ob.Conv
"""


def test_absent(package):
    assert run_python(LOAD, package.parent).stdout.startswith("None 0")


@pytest.mark.parametrize("content", ["cut", "text"])
def test_file_that_cannot_be_loaded(package, content):
    so = package / "_calls.so"
    if content == "cut":
        so.write_bytes(b"\x7fELF\x02\x01\x01" + bytes(57))
    else:
        so.write_text("not a library")
    out = run_python(LOAD, package.parent).stdout
    assert out.startswith("None 1") and "not used" in out


def test_other_torch(package):
    if not os.path.exists(os.path.join(PKG, "_calls.so")):
        pytest.skip("onnx-rs_b200/_calls.so is not built")
    os.symlink(os.path.join(PKG, "_calls.so"), package / "_calls.so")
    assert run_python(LOAD, package.parent).stdout.startswith("<module")
    out = run_python("import torch\ntorch.__version__ = '1.0.0'\n" + LOAD, package.parent).stdout
    assert out.startswith("None 1") and "1.0.0" in out


def test_first_seen_layout_loads_it(ob):
    """And without an operator of this path nothing does."""
    if not os.path.exists(os.path.join(PKG, "_calls.so")):
        pytest.skip("onnx-rs_b200/_calls.so is not built")
    run_python("""
import importlib, types, torch
ob = importlib.import_module("onnx-rs_b200")
op = ob.QuantizeBlocks()
op._describe = lambda h, x: (ob._capi.QuantizeDesc(), (((2,), (1,), torch.float32),) * 2, ())
assert "_calls" not in vars(ob.ops)
plan = op._described(types.SimpleNamespace(device=0), op._prepare, torch.zeros(3)).plan
assert plan is not None and "_calls.so" in open("/proc/self/maps").read()
""", ROOT)


def test_make_builds_it_again_for_another_python_or_torch(tmp_path):
    make = shutil.which("make")
    if not make:
        pytest.skip("no make")
    csrc = tmp_path / "pkg" / "csrc"
    csrc.mkdir(parents=True)
    shutil.copy(os.path.join(PKG, "csrc", "Makefile"), csrc)
    (csrc / "torch_calls.cpp").write_text("")
    version, log = tmp_path / "version", tmp_path / "log"
    python, cxx = tmp_path / "python", tmp_path / "cxx"
    python.write_text(f"#!/bin/sh\ncat {version}\n")
    cxx.write_text(f"#!/bin/sh\necho built >> {log}\ntouch ../_calls.so\n")
    for f in (python, cxx):
        f.chmod(0o755)
    for flags, builds in (("-DA", 1), ("-DA", 1), ("-DB", 2), ("-DB", 2)):
        version.write_text(flags + "\n")
        r = subprocess.run([make, "-s", "-C", str(csrc), "calls", f"PYTHON={python}", f"CXX={cxx}"], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        assert log.read_text().count("built") == builds
