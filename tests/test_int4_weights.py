"""4-bit weights as they are made: what a product that reads them at once finds, and values that no code stands for."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from omniasr_b200 import kernels

DEV = "cuda"


class Launches(TorchDispatchMode):
    """The memory that each operation's results lie in (views launch nothing)."""

    def __init__(self):
        super().__init__()
        self.written = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor) and not func.is_view and "empty" not in str(func) and "_unsafe_view" not in str(func):
            self.written.append(out.untyped_storage().data_ptr())
        return out


@pytest.mark.parametrize("n,k,group", [(8, 128, 128), (13, 160, 32), (64, 256, 64)])
def test_the_last_launch_writes_no_weights(n, k, group):
    """The products read weights before they wait for the launch before them, so that must not be one that writes them."""
    codes = torch.randint(0, 16, (n, k), dtype=torch.uint8)
    with Launches() as seen:
        w = kernels.int4_weights(codes, torch.ones(n, -(-k // group), dtype=torch.bfloat16), group)
    held = {w.codes.untyped_storage().data_ptr(), w.scales.untyped_storage().data_ptr()}
    assert len(held & set(seen.written)) == 2 and seen.written[-1] not in held
    with Launches() as seen:
        w = kernels.int4_quantise(torch.randn(n, k), group)
    assert seen.written[-1] not in {w.codes.untyped_storage().data_ptr(), w.scales.untyped_storage().data_ptr()}


def test_codes_that_are_none_are_refused():
    codes, scales = torch.full((9, 64), 15, dtype=torch.uint8), torch.ones(9, 1, dtype=torch.bfloat16)
    assert bool((kernels.int4_weights(codes, scales).values() == 7).all())
    codes[8, 63] = 16
    with pytest.raises(ValueError, match="code of 16"):
        kernels.int4_weights(codes, scales)


def test_weights_without_rows():
    w = kernels.int4_weights(torch.zeros(0, 64, dtype=torch.uint8), torch.ones(0, 2, dtype=torch.bfloat16), 32)
    assert w.values().shape == (0, 64)
    w = kernels.int4_quantise(torch.zeros(0, 160), 64)
    assert w.values().shape == (0, 160) and w.codes.shape == (0, 2, 512) and w.scales.shape == (0, 3, 8)


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
def test_groups_that_are_not_finite_are_nan(device):
    """A group with an infinity, a NaN or a number past float32's is NaN, its codes those of zeros; the others are as without it."""
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    want = kernels.int4_quantise(x.to(device), 32)
    bad = ((0, 3, float("nan")), (1, 40, float("inf")), (2, 70, float("-inf")), (3, 100, 1e300), (4, 127, float("inf")), (4, 126, float("-inf")))
    hide = torch.zeros(5, 4, dtype=torch.bool)
    for r, c, v in bad:
        x[r, c] = v
        hide[r, c // 32] = True
    w = kernels.int4_quantise(x.to(device), 32)
    wide = hide.repeat_interleave(32, 1)
    got = w.values().cpu()
    assert bool(got[wide].isnan().all()) and torch.equal(got[~wide], want.values().cpu()[~wide])
    unit = kernels.Int4Weights(w.codes, torch.ones_like(w.scales), w.n, w.k, w.group).values().cpu()
    assert bool((unit[wide] == 0).all())


@pytest.mark.gpu
def test_weights_made_just_before_in_a_graph():
    """Weights laid out and used in one graph, replayed over other codes: every product is that of the codes of its replay."""
    g = torch.Generator().manual_seed(0)
    codes, scales = torch.zeros(512, 1024, dtype=torch.uint8, device=DEV), torch.ones(512, 8, dtype=torch.bfloat16, device=DEV)
    x = torch.randint(-4, 5, (8, 1024), generator=g).bfloat16().to(DEV)
    step = lambda: kernels.decode_gemm_int4(x, kernels.int4_weights(codes, scales))  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = step()
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(20):
        codes.copy_(torch.randint(0, 16, codes.shape, generator=g, dtype=torch.uint8))
        graph.replay()
        want = (x.double() @ (codes.double() - 8).t()).bfloat16()  # (whole numbers: exact but for the one rounding)
        assert torch.equal(y, want)
