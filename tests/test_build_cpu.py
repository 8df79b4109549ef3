"""What `make` builds: the library with or without torch, and the tensor
operators again when Python or torch is another."""
import os
import stat
import subprocess

import pytest

from lcr_b200 import runtime as rt

TENSORS = os.path.join(rt.PKG_DIR, "csrc", "tensors.cpp")


def planned(python, *args):
    """The commands that a make would run with this Python."""
    p = subprocess.run(["make", "-n", "-C", rt.PKG_DIR, f"PYTHON={python}", *args], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    return p.stdout


def script(tmp_path, body):
    path = tmp_path / "python"
    path.write_text("#!/bin/sh\n" + body)
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return path


@pytest.mark.parametrize("body", ["exit 1\n", "echo 'No module named torch' >&2; exit 1\n"])
def test_a_make_without_torch_leaves_the_tensor_operators_out(tmp_path, body):
    out = planned(script(tmp_path, body), "-W", TENSORS)
    assert "tensors.cpp" not in out and "_tensors.so is left out" in out


def test_a_make_with_another_torch_builds_the_tensor_operators_again(tmp_path):
    python = script(tmp_path, "echo py399-torch99.0\n")
    assert "tensors.cpp" in planned(python)
