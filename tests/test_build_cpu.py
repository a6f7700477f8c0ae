"""What the build does again, and what it needs (make's own dry runs: nothing is compiled)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero_amd", "csrc")
pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def _would_run(*args):
    return subprocess.run(["make", "-n", "-C", CSRC, *args], check=True, capture_output=True, text=True).stdout


def test_changed_flags_rebuild_everything():
    out = _would_run("-W", "Makefile")
    for made in ("az_engine.hip -o az_engine.o", "az_tower.hip -o az_tower.o", "az_train.hip -o az_train.o", "-o libazamd.so", "az_torch.cpp -o ../network/_train_ops.so"):
        assert made in out, made


def test_every_kernel_is_built_without_packed_float32():
    for line in _would_run("-B").splitlines():
        if "hipcc" in line and " -c " in line:
            assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line


def test_build_compiles_what_is_already_there():
    """build() is the check that the sources compile, so it does not go by the age of what was built before."""
    import __graft_entry__ as g
    ran = []

    class Stop(Exception):
        pass

    def note(cmd):
        ran.append(cmd)
        raise Stop
    real, g.subprocess.check_call = g.subprocess.check_call, note
    try:
        with pytest.raises(Stop):
            g.build()
    finally:
        g.subprocess.check_call = real
    assert ran[0][0] == "make" and "-B" in ran[0]


def test_the_c_library_needs_no_pytorch(tmp_path):
    """With a Python that has no PyTorch, or without a Python, libazamd.so is all that is built, and nothing fails."""
    bare = tmp_path / "python"
    bare.write_text("#!/bin/sh\nexec %s -S -E \"$@\"\n" % shutil.which("python3"))
    bare.chmod(0o755)
    for python in (str(bare), str(tmp_path / "no-such-python")):
        out = _would_run("-B", "PYTHON=" + python)
        assert "-o libazamd.so" in out and "_train_ops" not in out
    assert "-o ../network/_train_ops.so" in _would_run("-B")


def test_another_pytorch_rebuilds_the_binding():
    import torch
    out = _would_run("-W", os.path.join(os.path.dirname(torch.__file__), "version.py"))
    assert "az_torch.cpp -o ../network/_train_ops.so" in out
