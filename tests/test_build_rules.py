"""The kernel library's build rules (CPU: make's dry run)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eventstreamgpt_amd", "csrc")


def test_a_change_of_the_flags_rebuilds_every_object():
    """The flags stand in the Makefile: were it newer than the objects, each of them and both libraries would be made again
    (objects of two sets of flags must not be linked together)."""
    if shutil.which("make") is None:
        pytest.skip("no make")
    run = subprocess.run(["make", "-n", "-C", CSRC, "-W", "Makefile"], capture_output=True, text=True, check=True)
    lines = run.stdout.splitlines()
    sources = [f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")) and f != "torch_ops.cpp"]
    for f in sources:
        assert any(" -c " + f + " " in line for line in lines), f
    assert any("-o ../libesgpt_amd.so" in line for line in lines)
    assert any("torch_ops.cpp" in line and "-o ../libesgpt_torch.so" in line for line in lines)
