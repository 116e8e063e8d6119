"""Calls with tensors of a device that is not the current one, without a GPU: the library is replaced by a recorder of what is
current when it is reached."""

import contextlib
import os
import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from omniasr_b200 import kernels


@pytest.fixture
def gpus(monkeypatch):
    """Two GPUs that are names alone; ``state.current`` is the current one."""
    state = types.SimpleNamespace(current=0, seen=[])

    @contextlib.contextmanager
    def device(d):
        before, state.current = state.current, torch.device(d).index
        try:
            yield
        finally:
            state.current = before

    monkeypatch.setattr(kernels, "_current", lambda: state.current)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(kernels, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(kernels, "_status", {i: torch.zeros(1, dtype=torch.int32) for i in range(2)})
    return state


def on(index, **more):
    return types.SimpleNamespace(device=torch.device("cuda", index), dtype=torch.bfloat16, **more)


@pytest.mark.parametrize("index", [0, 1])
def test_paged_and_packed_calls_run_on_their_tensors_device(gpus, monkeypatch, index):
    def record(name):
        return lambda *args: gpus.seen.append((name, gpus.current))

    names = ["paged_rope_kv", "paged_kv_read", "paged_attention", "packed_attention"]
    monkeypatch.setattr(kernels, "_binding", lambda: types.SimpleNamespace(**{n: record(n) for n in names}))
    t = on(index)
    kernels.paged_rope_kv(t, t, t, t, t, t, 1, 1)
    kernels.paged_kv_read(t, t, t, t, 1)
    kernels.paged_attention(t, t, t, t, t, 1.0)
    kernels.packed_attention(t, t, t, t)
    kernels.packed_attention(k=t, v=t, q_offsets=t, q=t)
    assert gpus.seen == [(n, index) for n in names + ["packed_attention"]]
    assert gpus.current == 0


def test_the_current_device_is_put_back_after_an_error(gpus, monkeypatch):
    def refuse(*args):
        assert gpus.current == 1
        raise ValueError("no")

    monkeypatch.setattr(kernels, "_binding", lambda: types.SimpleNamespace(packed_attention=refuse))
    with pytest.raises(ValueError, match="no"):
        kernels.packed_attention(*[on(1)] * 4)
    assert gpus.current == 0


def test_every_call_of_the_library_is_guarded():
    """The other public functions take the guard as well: each is the wrapper around the function that it names."""
    names = ["rope_kv", "decode_attention", "draft_attention", "beam_attention", "prefill_attention", "prefill_attention_grouped",
             "propose", "accept", "beam_select", "decode_gemm", "decode_gemm_rope", "reorder_gather"]
    for n in names:
        fn = getattr(kernels, n)
        assert fn.__wrapped__.__name__ == n and fn.__doc__ == fn.__wrapped__.__doc__


def test_import_without_cuda_in_pytorch():
    """A build of PyTorch without CUDA has none of the private CUDA functions: the package still imports, and says that no
    device is available."""
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "from omniasr_b200 import kernels\n"
            "assert not kernels.available(torch.device('cpu'))\n")
    root = Path(kernels.__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": str(root)}, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
