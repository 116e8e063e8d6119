"""Kernels that start before the kernel before them has ended read what that one may write by ordinary loads only."""

import re

from conftest import ROOT

CSRC = ROOT / "omniasr-trt_b200" / "csrc"
# Loads through the read-only path that stay, with the lines that have them: weights, which no kernel of the stream writes.
ALLOWED = {"wgemm4.cu": {"__ldg(s0", "__ldg(s1"}}


def test_no_read_only_loads_of_what_earlier_kernels_write():
    """A file counts if its kernels are launched early, or if it is included (headers)."""
    seen = 0
    for path in sorted(CSRC.glob("*.cu*")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        if path.suffix == ".cu" and "launch_dependent" not in text and "griddepcontrol" not in text:
            continue
        seen += 1
        for m in re.finditer(r"__ldg\s*\(\s*\w*|ld\.global(\.\w+)*\.nc|const \w+\s*\*\s*__restrict__", text):
            call = re.sub(r"\s", "", m.group()) if m.group().startswith("__ldg") else m.group()
            if path.name == "attention.cu" and "__restrict__" in call:
                continue  # combine_kernel, launched in order
            assert call in ALLOWED.get(path.name, ()), f"{path.name}: {call}"
    assert seen > 10
