"""The operators of a 4-bit serving step together: the example with a 4-bit cache, 4-bit weights, norms of queries and keys, and the
decode loop as a graph over tables on the GPU, against the same loop steered by the host; and a step's calls on their own streams,
devices' tables and captures."""

import sys

import pytest
import torch

import int4_util as iu
from conftest import ROOT
from omniasr_b200 import kernels
from omniasr_b200.paged import Batch, DeviceTables, PagedCache

DEV = "cuda"


def example():
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import paged_serving
    finally:
        sys.path.pop(0)
    return paged_serving


def test_tables_refuse_and_hand_over_pages():
    cache = PagedCache(1, 10, 8, 1, 32, kind=torch.uint8, device="cpu")
    assert cache.k.shape == (1, 10, 1, 8, 16) and cache.k_scale.shape == (1, 10, 1, 8, 1)
    s = cache.add()
    cache.extend([s], [17])
    t = cache.device_tables(3, 4, 5)
    assert cache.free_pages == 2 and t.free.tolist() == [7, 6, 5, 4, 3] and int(t.free_count) == 5
    with pytest.raises(ValueError, match="device_tables"):
        cache.device_tables(3, 4, 3)
    with pytest.raises(ValueError, match="tokens"):
        t.plan(torch.arange(2), torch.ones(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="4-bit"):
        PagedCache(1, 10, 8, 1, 16, kind=torch.uint8, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 8), (2, 2, 512, 64)])
@pytest.mark.parametrize("kind,norms,int4", [(torch.uint8, True, True), (torch.uint8, False, False), (torch.bfloat16, True, False)])
def test_graphed_loop_gives_the_hosts_tokens(heads, kv, dim, page, kind, norms, int4):
    ps = example()
    model = ps.Decoder(heads=heads, kv_heads=kv, dim=dim, norms=norms, int4=int4)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 200, 1, 63, 64)]
    host = ps.serve(model, prompts, 8, kind, page=page, chunk=256)
    graph = ps.serve(model, prompts, 8, kind, page=page, graph=True)
    assert host == graph and all(len(o) == 9 for o in host)
    assert kernels.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.uint8, torch.float8_e4m3fn, torch.bfloat16])
def test_a_refused_request_leaves_the_others_alone(kind):
    """Pages for three of four requests: the others' rows are written and attended as without it, its sequence stays as it was."""
    heads, kv, dim, page = 4, 2, 64, 8
    g = torch.Generator().manual_seed(2)
    cs = torch.ones(64, dim // 2, 2, device=DEV)
    cs[..., 1] = 0
    qkv = torch.randn(4 * 9, (heads + 2 * kv) * dim, generator=g).bfloat16().to(DEV)
    rows = torch.arange(4, device=DEV)
    got = []
    for pages in (4 * 2, 3 * 2):
        cache = PagedCache(1, pages, page, kv, dim, kind=kind)
        tables = cache.device_tables(4, 2)
        batch = tables.plan(rows, 9)
        o = cache.decode(0, qkv, cs, batch, heads)
        got.append((batch.taken.tolist(), tables.length.tolist(), o.view(4, 9, heads, dim), int(tables.free_count)))
    assert got[0][0] == [True] * 4 and got[1][0] == [True, True, True, False]
    assert got[1][1] == [9, 9, 9, 0] and got[1][3] == 0
    assert torch.equal(got[0][2][:3], got[1][2][:3])
    assert kernels.read_status() == 0


@pytest.mark.gpu
def test_two_captured_steps_and_an_eager_one():
    """Two graphs of 4-bit attention captured on one stream, replayed in turn with an eager call between: each gives what it gave."""
    g = torch.Generator().manual_seed(4)
    heads, kv, dim, page = 8, 2, 128, 16
    k, v, ks, vs, kval, vval = (t.to(DEV) for t in iu.cache(40, kv, page, dim, g))
    table = torch.randperm(40, generator=g).to(torch.int32).view(2, 20).to(DEV)
    lens = [torch.tensor([300, 17], device=DEV), torch.tensor([5, 320], device=DEV)]
    q = torch.randn(2, heads, dim, generator=g).bfloat16().to(DEV)
    call = lambda i: kernels.paged_attention(q, k, v, table, lens[i], 0.1, k_scale=ks, v_scale=vs)  # noqa: E731
    want = [call(0).clone(), call(1).clone()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graphs, outs = [], []
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(call(i))
            graphs.append(graph)
        for _ in range(3):
            for i in (0, 1, 1, 0):
                graphs[i].replay()
                eager = call(i)
                assert torch.equal(outs[i], want[i]) and torch.equal(eager, want[i])
    torch.cuda.current_stream().wait_stream(stream)
    assert kernels.read_status() == 0


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams do not share what they work in."""
    g = torch.Generator().manual_seed(5)
    k, v, ks, vs, _, _ = (t.to(DEV) for t in iu.cache(300, 2, 16, 128, g))
    table = torch.randperm(300, generator=g).to(torch.int32).view(3, 100).to(DEV)
    length = torch.tensor([1500, 900, 1600], device=DEV)
    q = torch.randn(3, 16, 128, generator=g).bfloat16().to(DEV)
    state = lambda: DeviceTables(3, 100, 16, list(range(300)))  # noqa: E731
    want = kernels.paged_attention(q, k, v, table, length, 0.1, k_scale=ks, v_scale=vs)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, plans, tables = [[], []], [[], []], [state(), state()]
    rows = torch.arange(3, device=DEV)
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(kernels.paged_attention(q, k, v, table, length, 0.1, k_scale=ks, v_scale=vs))
                plans[i].append(tables[i].plan(rows, 7))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for side in outs for o in side)
    for a, b in zip(*plans):
        assert torch.equal(a.slots, b.slots) and torch.equal(a.table, b.table) and bool(a.taken.all())
    assert tables[0].length.tolist() == [140] * 3
    assert kernels.read_status() == 0


def test_prefill_needs_the_number_of_keys():
    cache = PagedCache(1, 4, 8, 1, 32, kind=torch.uint8, device="cpu")
    none = torch.zeros(0)
    batch = Batch(2, [2], None, none, none, none, none, none, none, False, none)
    with pytest.raises(ValueError, match="total"):
        cache.prefill(0, none, none, batch, 1)
