"""The build's commands, without running them."""

import subprocess
import sys
from pathlib import Path

import __graft_entry__ as entry

CSRC = Path(entry.__file__).resolve().parent / "omniasr-trt_b200" / "csrc"


def test_the_extension_is_built_for_this_interpreter(monkeypatch):
    """build() names its own interpreter to make, and make asks that one for PyTorch's paths."""
    seen = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: seen.append(cmd))
    monkeypatch.setattr(entry, "install_reference", lambda: "absent")
    entry.build()
    assert seen[0][0] == "make" and f"PYTHON={sys.executable}" in seen[0]
    assert "$(PYTHON) -c" in (CSRC / "Makefile").read_text()


def test_the_c_library_builds_without_pytorch():
    """`make lib` runs no python and touches no PyTorch header."""
    r = subprocess.run(["make", "-C", str(CSRC), "-n", "-B", "lib", "PYTHON=/nonexistent/python"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "libomniasr_b200.so" in r.stdout and "torch" not in r.stdout and "nonexistent" not in r.stderr
