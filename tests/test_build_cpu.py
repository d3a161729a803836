"""What `make` in csrc/ builds: the C ABI's libraries without torch, the host module where torch is, and again where it is another one."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "selfc_amd", "csrc")

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="needs make")


def plan(*args, cwd=CSRC):
    """the commands that make would run"""
    return subprocess.run(["make", "-n", *args], cwd=cwd, check=True, capture_output=True, text=True).stdout


def test_without_torch_the_libraries_are_all(tmp_path):
    bare = tmp_path / "python"                              # an interpreter that has no torch
    bare.write_text('#!/bin/sh\necho ""\n')
    bare.chmod(0o755)
    out = plan("-B", f"PYTHON={bare}")
    assert "libselfc_hip.so" in out and "libselfc_hip_bf16.so" in out and "host.cpp" not in out
    assert "host.cpp" not in plan("-B", "libs")
    assert "host.cpp" in plan("-B")


def test_another_torch_builds_the_host_module_again(tmp_path):
    csrc = tmp_path / "selfc_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    shutil.copy(os.path.join(CSRC, "Makefile"), csrc)
    (csrc / "host.cpp").write_text("")
    (tmp_path / "include" / "selfc_hip.h").write_text("")
    torch = tmp_path / "site" / "torch"
    torch.mkdir(parents=True)
    (torch / "__init__.py").write_text("")
    (torch / "version.py").write_text("1")
    made = lambda: "host.cpp" in subprocess.run(["make", "../_host.so", "CXX=touch ../_host.so #"], cwd=csrc, check=True, capture_output=True, text=True,  # noqa: E731
                                                env=dict(os.environ, PYTHONPATH=str(tmp_path / "site"))).stdout
    assert made() and not made()
    (torch / "version.py").write_text("2")
    assert made() and not made()
