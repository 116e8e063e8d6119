"""The attention calls' workspaces, on the CPU."""

import pytest
import torch

from omniasr_b200 import kernels


@pytest.fixture
def empty(monkeypatch):
    monkeypatch.setattr(kernels, "_ATTN_WS", {})
    monkeypatch.setattr(kernels, "_ATTN_WS_RETIRED", [])


def test_outgrown_workspaces_stay_few(empty):
    """Calls that each need a little more than the one before: the workspaces kept for captured graphs are few and together
    no more than twice the last."""
    device = torch.device("cpu")
    for n in range(1 << 20, 1 << 24, 9973):
        ws = kernels._attn_workspace(n, device, 0)
        assert ws.numel() >= n and int(ws[:64].sum()) == 0
        assert kernels._attn_workspace(n, device, 0) is ws
    assert len(kernels._ATTN_WS_RETIRED) <= 8
    assert sum(t.numel() for t in kernels._ATTN_WS_RETIRED) <= 2 * ws.numel()
    assert ws.numel() <= 1.5 * (1 << 24)


def test_streams_have_their_own(empty):
    device = torch.device("cpu")
    a, b = kernels._attn_workspace(100, device, 1), kernels._attn_workspace(100, device, 2)
    assert a is not b and kernels._attn_workspace(100, device, 1) is a
