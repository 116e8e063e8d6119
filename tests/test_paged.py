"""The paged cache and the packed-prompt attention without a GPU: argument checks, and the plain forms in 64 bits that the
GPU tests compare with, checked against each other and against differently written ones."""

import pytest
import torch

import paged_util as pu
from omniasr_b200 import kernels


def test_oracle_quantisation_matches_its_definition():
    """e is the smallest integer with max|x| <= 448 * 2^e, the codes lie within half a step of x * 2^-e."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 64, generator=g) * torch.exp(6 * torch.randn(200, 1, generator=g))
    x[0] = 0
    codes, e = pu.quantise(x)
    amax = x.abs().amax(-1).double()
    top = 448.0 * 2.0 ** e.double()
    assert bool((amax <= top).all())
    live = (e > -40) & (e < 40)
    assert bool((amax[live] > top[live] / 2).all())
    back = pu.dequantise(codes, (e + 127).to(torch.uint8)).double()
    # e4m3: 3 fraction bits (half a step is 2^-4 of the value), below 2^-6 a fixed step of 2^-9.
    bound = torch.maximum(x.double().abs() * 2.0**-4, 2.0 ** (e.double()[:, None] - 10))
    assert bool(((back - x.double()).abs() <= bound).all())


def test_oracle_paged_equals_packed():
    """A row of T new tokens over its pages is a packed sequence of T queries and all its keys."""
    g = torch.Generator().manual_seed(1)
    t, heads, kv, dim, page = 3, 6, 2, 16, 4
    lens = [0, 1, 7, 8]
    k = torch.randn(12, kv, page, dim, generator=g, dtype=torch.float64)
    v = torch.randn(12, kv, page, dim, generator=g, dtype=torch.float64)
    table = torch.randperm(12, generator=g).view(4, 3)
    q = torch.randn(4 * t, heads, dim, generator=g, dtype=torch.float64)
    want = pu.paged(q, k, v, table, torch.tensor(lens), 0.3, t)
    ks, vs = [], []
    for r, n in enumerate(lens):
        ids = table[r]
        ks.append(k[ids].transpose(1, 2).reshape(-1, kv, dim)[: n + t - 1])
        vs.append(v[ids].transpose(1, 2).reshape(-1, kv, dim)[: n + t - 1])
    k_off = [0]
    for n in lens:
        k_off.append(k_off[-1] + n + t - 1)
    got = pu.packed(q, torch.cat(ks), torch.cat(vs), [0, t, 2 * t, 3 * t, 4 * t], k_off, 0.3)
    assert torch.allclose(got, want, atol=1e-12)
    assert bool((want[0] == 0).all())  # row 0's first query sees nothing


def _pages(dtype=torch.bfloat16, pages=4, kv=2, page=8, dim=64):
    return torch.zeros(pages, kv, page, dim, dtype=dtype), torch.zeros(pages, kv, page, dim, dtype=dtype)


def test_argument_checks():
    """What the wrappers refuse before any kernel is reached."""
    k, v = _pages()
    table = torch.zeros(2, 2, dtype=torch.int32)
    lengths = torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    att = lambda **kw: kernels.paged_attention(**{**dict(q=q, k_pages=k, v_pages=v, page_table=table, lengths=lengths,
                                                         scale=1.0), **kw})  # noqa: E731
    with pytest.raises(ValueError, match="dtype"):
        att(q=q.half())
    with pytest.raises(ValueError, match="supported"):
        att(k_pages=k.float(), v_pages=v.float())
    with pytest.raises(ValueError, match="strides"):
        att(v_pages=v.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="scales"):
        att(k_scale=torch.zeros(4, 2, 8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="uint8 scales"):
        k8, v8 = _pages(torch.float8_e4m3fn)
        att(k_pages=k8, v_pages=v8)
    with pytest.raises(ValueError, match="int32"):
        att(page_table=table.long())
    with pytest.raises(ValueError, match="tokens"):
        att(tokens=2)
    with pytest.raises(ValueError, match="head_dim"):
        att(q=torch.zeros(2, 4, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        att(q=torch.zeros(2, 64, 4, dtype=torch.bfloat16).transpose(1, 2))
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    cs = torch.zeros(16, 32, 2)
    idx = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="qkv"):
        kernels.paged_rope_kv(qkv, cs, idx, k, v, idx, 5, 2)
    with pytest.raises(ValueError, match="per token"):
        kernels.paged_rope_kv(qkv, cs, idx[:2], k, v, idx, 4, 2)
    with pytest.raises(ValueError, match="cs"):
        kernels.paged_rope_kv(qkv, cs[:, :16], idx, k, v, idx, 4, 2)
    with pytest.raises(ValueError, match="dtype"):
        kernels.paged_kv_read(k, v, table, torch.zeros(3, dtype=torch.int64), 0, dtype=torch.float16)
    with pytest.raises(ValueError, match="page_table"):
        kernels.paged_kv_read(k, v, table, torch.zeros(4, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="share a dtype"):
        kernels.packed_attention(q, q.float(), q.float(), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="sequences"):
        kernels.packed_attention(q, q, q, torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="unit stride"):
        kernels.packed_attention(q, q.transpose(1, 2).contiguous().transpose(1, 2), q.transpose(1, 2).contiguous().transpose(1, 2),
                                 torch.zeros(2, dtype=torch.int64))


def test_workspace_sizes():
    from omniasr_b200 import _lib

    lib = _lib.load()
    size = lib.omniasr_paged_attention_workspace
    assert size(_lib.F32, _lib.F32, 4, 1, 8, 2, 64, 16, 100) >= 65536 + 4 * 8 * 66 * 4  # counters, one split at least
    assert size(_lib.BF16, _lib.FP8, 4, 1, 8, 2, 128, 16, 100) > 65536
    assert size(_lib.BF16, _lib.BF16, 4, 1, 8, 3, 128, 16, 100) == 0  # heads not a multiple
    assert size(_lib.BF16, _lib.BF16, 4, 1, 8, 2, 96, 16, 100) == 0  # head_dim


def test_paged_cache_hands_out_pages():
    """Pages, slots and offsets of a batch; nothing changes when the pages do not suffice; freed pages come back."""
    from omniasr_b200.paged import PagedCache

    c = PagedCache(2, 7, 4, 2, 16, device="cpu")
    a, b = c.add(), c.add()
    step = c.extend([a, b], [5, 0])
    assert step.tokens == 5 and step.total == 5 and step.fresh
    assert step.pos.tolist() == [0, 1, 2, 3, 4]
    assert step.lengths.tolist() == [1, 1]
    assert step.q_offsets.tolist() == [0, 5, 5] == step.k_offsets.tolist()
    pages = step.table[0].tolist()
    assert len(set(pages)) == 2
    assert step.slots.tolist() == [pages[0] * 4 + i for i in range(4)] + [pages[1] * 4]
    step = c.extend([b, a], [9, 4])
    assert step.pos.tolist() == [*range(9), 5, 6, 7, 8]
    assert step.k_offsets.tolist() == [0, 9, 18] and step.lengths.tolist() == [1, 6] and not step.fresh
    assert sorted(set(step.table[0].tolist()) | set(step.table[1].tolist())) == sorted(set(range(7)) - set(c._free))
    assert len(set((step.slots).tolist())) == 13
    with pytest.raises(RuntimeError, match="full"):
        c.extend([a, b], [4, 8])
    assert c.length(a) == 9 and c.length(b) == 9 and c.free_pages == 1
    with pytest.raises(ValueError, match="different"):
        c.extend([a, a], [1, 1])
    c.free(a)
    assert c.free_pages == 4
    assert c.extend([b], [3]).total == 12
    c.free(b)
    assert c.free_pages == 7


def test_paged_cache_drops_drafts():
    from omniasr_b200.paged import PagedCache

    c = PagedCache(1, 5, 4, 1, 16, device="cpu")
    a = c.add()
    pages = c.extend([a], [7]).table[0].tolist()
    c.extend([a], [6])  # to 13 positions: two more pages
    assert c.free_pages == 1
    c.trim(a, 8)  # the first 8 fill two pages
    assert c.length(a) == 8 and c.free_pages == 3
    step = c.extend([a], [1])
    assert step.table[0, :2].tolist() == pages and step.pos.tolist() == [8] and step.lengths.tolist() == [9]
    for n in (-1, 10):
        with pytest.raises(ValueError, match="trim"):
            c.trim(a, n)
    c.trim(a, 0)
    assert c.free_pages == 5 and c.extend([a], [1]).fresh


def test_paged_cache_decode_wants_even_steps():
    from omniasr_b200.paged import PagedCache

    c = PagedCache(1, 4, 4, 1, 16, device="cpu")
    batch = c.extend([c.add(), c.add()], [1, 2])
    with pytest.raises(ValueError, match="same number"):
        c.decode(0, torch.zeros(3, 48), torch.zeros(8, 8, 2), batch, 1)
