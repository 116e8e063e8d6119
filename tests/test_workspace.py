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


def test_captures_have_their_own(empty, monkeypatch):
    """What a capture allocates is zeroed inside it: another capture on the stream, and eager calls, get others."""
    capture = 0
    monkeypatch.setattr(kernels, "_capture_id", lambda stream: capture)
    monkeypatch.setattr(kernels, "_CAPTURE_WS", {})
    device = torch.device("cpu")
    capture = 7
    a = kernels._attn_workspace(100, device, 1)
    assert kernels._attn_workspace(100, device, 1) is a
    bigger = kernels._attn_workspace(3 << 20, device, 1)
    assert bigger.numel() >= 3 << 20 and kernels._attn_workspace(100, device, 1) is bigger
    capture = 8
    b = kernels._attn_workspace(100, device, 1)
    assert b is not a and b is not bigger
    capture = 0
    c = kernels._attn_workspace(100, device, 1)
    assert c is not b and kernels._attn_workspace(100, device, 1) is c
    capture = 9  # one that eager calls have zeroed serves captures as well
    assert kernels._attn_workspace(100, device, 1) is c
    assert kernels._ATTN_WS_RETIRED == []


@pytest.mark.gpu
def test_graphs_captured_before_any_is_replayed():
    """Two graphs of a step on a stream without a workspace; the second is replayed alone, then the first, then an eager call."""
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(40, 2, 16, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([633], device="cuda")
    q = torch.randn(1, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    x = torch.randn(633, 2, 128, generator=g, device="cuda").to(torch.bfloat16)
    qp = torch.randn(70, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    off, k_off = torch.tensor([0, 70], device="cuda"), torch.tensor([0, 633], device="cuda")

    def step():
        return kernels.paged_attention(q, k, v, table, lengths, 0.1), kernels.packed_attention(qp, x, x, off, k_off)

    want = step()
    torch.cuda.synchronize()
    stale = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")  # what fresh memory may hold
    del stale
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        graphs.append((graph, out))
    for graph, out in reversed(graphs):
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.cuda.stream(side):
        out = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert kernels.read_status() == 0
