"""Requests that tables on the GPU refuse, beside others: in steps of prompts and of single tokens, with rope tables as long as the
tables are.

Attention of the others is compared with that of a step without the refused ones, whose work is cut otherwise: each side is within
2^-8 |o| + (2^-8 + 2^-10) A of the formula's o (the bound of test_paged_gpu.py; 4-bit pages' is smaller), |o| and A = sum p |v| / sum p are at
most the largest |v|, so they are at most 2 (2^-7 + 2^-10) of that apart."""

import pytest
import torch

from omniasr_b200 import kernels
from omniasr_b200.paged import PagedCache

pytestmark = pytest.mark.gpu

DEV = "cuda"
HEADS, KV, DIM, PAGE = 4, 2, 64, 8


def rope(positions):
    angle = torch.arange(positions)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2) / DIM)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(DEV)


def close(a, b, v):
    """v: the values that either side may see."""
    return bool(((a.float() - b.float()).abs() <= 2 * (2.0**-7 + 2.0**-10) * float(v.abs().max())).all())


def qkv_of(n, seed):
    return torch.randn(n, (HEADS + 2 * KV) * DIM, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("kind", [torch.uint8, torch.float8_e4m3fn, torch.bfloat16])
def test_positions_past_the_tables_are_no_bad_index(kind, norms):
    """A sequence that fills its table row and asks for more is refused without a status, here and in the append."""
    width, cs = 2, rope(2 * PAGE)
    w = (torch.ones(DIM, dtype=torch.bfloat16, device=DEV),) * 2 + (1e-6,) if norms else None
    cache = PagedCache(1, 8, PAGE, KV, DIM, kind=kind)
    tables = cache.device_tables(3, width)
    rows = torch.arange(3, device=DEV)
    new = torch.tensor([5, 16, 9], device=DEV)
    batch = tables.plan(rows, new, 30, total=30)
    cache.prefill(0, qkv_of(30, 0), cs, batch, HEADS, norms=w)
    assert kernels.read_status() == 0
    held = [cache.k.clone(), cache.v.clone()]
    batch = tables.plan(rows, 2)
    assert batch.taken.tolist() == [True, False, True] and tables.length.tolist() == [7, 16, 11]
    o = cache.decode(0, qkv_of(6, 1), cs, batch, HEADS, norms=w).view(3, 2, HEADS, DIM)
    assert kernels.read_status() == 0
    # the refused sequence's pages are as they were, the others' rows those of a step without it
    full = tables.table[1].long()
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    assert torch.equal(raw(cache.k)[0][full], raw(held[0])[0][full]) and torch.equal(raw(cache.v)[0][full], raw(held[1])[0][full])
    tables.trim(rows, torch.tensor([5, 16, 9], device=DEV))
    two = torch.tensor([0, 2], device=DEV)
    batch = tables.plan(two, 2)
    alone = cache.decode(0, qkv_of(6, 1).view(3, 2, -1)[[0, 2]].reshape(4, -1), cs, batch, HEADS, norms=w).view(2, 2, HEADS, DIM)
    assert close(o[[0, 2]], alone, torch.cat([qkv_of(30, 0), qkv_of(6, 1)])[:, -KV * DIM:])
    assert kernels.read_status() == 0


@pytest.mark.parametrize("kind", [torch.uint8, torch.float8_e4m3fn, torch.bfloat16])
def test_a_refused_prompt_leaves_the_others_alone(kind):
    """A prompt for which there are no pages, and one past its table row: queries without keys of their own between the others'."""
    cs = rope(6 * PAGE)
    new = [20, 33, 7, 60, 12]  # the second finds too few pages (3 + 5 + 1 + 2 > 7), the fourth passes the table
    n = sum(new)
    qkv = qkv_of(n, 2)
    cache = PagedCache(1, 7, PAGE, KV, DIM, kind=kind)
    tables = cache.device_tables(5, 6)
    rows = torch.arange(5, device=DEV)
    batch = tables.plan(rows, torch.tensor(new, device=DEV), n, total=n)
    assert batch.taken.tolist() == [True, False, False, False, False]  # (those behind one that waits for pages wait too)
    o = cache.prefill(0, qkv, cs, batch, HEADS)
    assert kernels.read_status() == 0 and bool(torch.isfinite(o[:20]).all())
    alone = PagedCache(1, 7, PAGE, KV, DIM, kind=kind)
    a = alone.add()
    assert close(o[:20], alone.prefill(0, qkv[:20], cs, alone.extend([a], [20]), HEADS), qkv[:20, -KV * DIM:])
    # a sequence with keys whose chunk is refused: its queries outnumber its keys
    chunk = torch.tensor([3, 40, 4], device=DEV)
    some = torch.tensor([1, 0, 2], device=DEV)
    batch = tables.plan(some, chunk, 47, total=64)
    assert batch.taken.tolist() == [True, False, True] and tables.length.tolist() == [20, 3, 4, 0, 0]
    got = cache.prefill(0, qkv_of(47, 3), cs, batch, HEADS)
    assert kernels.read_status() == 0
    other = PagedCache(1, 7, PAGE, KV, DIM, kind=kind)
    b, c = other.add(), other.add()
    part = qkv_of(47, 3)
    want = other.prefill(0, torch.cat([part[:3], part[43:]]), cs, other.extend([b, c], [3, 4]), HEADS)
    assert close(torch.cat([got[:3], got[43:]]), want, part[:, -KV * DIM:])


def test_positions_must_be_some():
    state = tuple(t.to(DEV) for t in (torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int32), torch.arange(5, dtype=torch.int32),
                                      torch.full((1,), 5)))
    rows, new = torch.tensor([1, 2], device=DEV), torch.tensor([40, 3], device=DEV)
    for bad in (0, -5):
        with pytest.raises(ValueError, match="positions"):
            kernels.paged_plan(rows, new, 43, 8, *state, positions=bad)
    pos, slots, *_, taken = kernels.paged_plan(rows, new, 43, 8, *state, positions=10)  # (taken tokens' positions are what they are)
    assert taken.tolist() == [False, True] and pos.tolist() == [min(i, 9) for i in range(40)] + [0, 1, 2]
    assert bool((slots[:40] == -1).all()) and kernels.read_status() == 0
