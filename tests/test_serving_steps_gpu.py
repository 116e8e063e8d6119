"""The serving example for every small number of steps: as a graph it gives what the loop that the host steers gives."""

import sys

import pytest
import torch

from conftest import ROOT
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [0, 1, 2])
def test_steps(steps):
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import paged_serving as ps
    finally:
        sys.path.pop(0)
    model = ps.Decoder()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 64, 1)]
    host = ps.serve(model, prompts, steps, torch.uint8, chunk=256)
    graph = ps.serve(model, prompts, steps, torch.uint8, graph=True)
    assert all(len(o) == 1 + steps for o in host) and graph == host
    assert kernels.read_status() == 0
