"""What the library does once per device (csrc/per_device.h), compiled for the host."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "omniasr-trt_b200" / "csrc"

MAIN = r"""
#include <assert.h>
#include "per_device.h"
int main() {
  omni::PerDevice d;
  int calls = 0, answer = 0;
  auto set = [&] { ++calls; return answer; };
  assert(d.once(0, set) == 0 && calls == 1);
  assert(d.once(0, set) == 0 && calls == 1);   // done for device 0
  assert(d.once(1, set) == 0 && calls == 2);   // not for device 1
  assert(d.once(1, set) == 0 && d.once(0, set) == 0 && calls == 2);
  answer = 7;
  assert(d.once(63, set) == 7 && calls == 3);  // a failure is given back and not taken for done
  assert(d.once(63, set) == 7 && calls == 4);
  answer = 0;
  assert(d.once(63, set) == 0 && d.once(63, set) == 0 && calls == 5);
  assert(d.once(64, set) == 0 && d.once(64, set) == 0 && d.once(-1, set) == 0 && calls == 8);
}
"""


def test_once_per_device(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "main.cpp"
    src.write_text(MAIN)
    subprocess.run([cxx, "-std=c++17", "-I", str(CSRC), str(src), "-o", str(tmp_path / "main")], check=True)
    subprocess.run([str(tmp_path / "main")], check=True)


def test_no_launcher_keeps_one_flag_for_all_devices():
    """Every kernel that takes more than the default shared memory asks for it per device."""
    for f in CSRC.glob("*.cu"):
        text = f.read_text()
        assert "cudaFuncSetAttribute" not in text, f"{f.name}: allow_smem() sets it per device"
