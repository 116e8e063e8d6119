"""Packed attention where keys or values are not ordinary numbers: scores that are NaN or +inf, hidden values that are NaN,
infinite or the type's largest, one NaN in a long sequence.

Tolerances as in test_paged_gpu: bf16 outputs and probabilities of 8 significant bits, 2^-8 (|o| + A) with A = sum p |v| / sum p,
and 2^-10 A for the exponential and the fp32 sums. References are float64, by masked matrix products on the GPU."""

import time

import pytest
import torch

from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAN, INF = float("nan"), float("inf")


def randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV).to(torch.bfloat16)


def offsets(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def packed(q, k, v, new, keys, scale=None):
    return kernels.packed_attention(q, k, v, torch.tensor(offsets(new), device=DEV), torch.tensor(offsets(keys), device=DEV), scale)


def plain(q, k, v, new, keys, scale=None):
    """(o, A) in float64; keys that a query does not see take no part (k and v finite)."""
    heads, kv, dim = q.size(1), k.size(1), q.size(2)
    scale = dim**-0.5 if scale is None else scale
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for a, b, c, d in zip(offsets(new), offsets(new)[1:], offsets(keys), offsets(keys)[1:]):
        if b == a or d == c:
            continue
        seen = torch.arange(1, b - a + 1, device=DEV) + (d - c) - (b - a)
        mask = torch.arange(d - c, device=DEV)[None] >= seen[:, None]
        for h in range(heads):
            j = h // (heads // kv)
            x = (q[a:b, h].double() @ k[c:d, j].double().t() * scale).masked_fill(mask, -INF)
            p = torch.nan_to_num(torch.softmax(x, -1))  # (a query that sees nothing: zeros)
            out[a:b, h], size[a:b, h] = p @ v[c:d, j].double(), p @ v[c:d, j].double().abs()
    return out, size


def check(got, want, size):
    bound = 2.0**-8 * (want.abs() + size) + 2.0**-10 * size + 1e-30
    got = got.double()
    assert bool(torch.isfinite(got).all()), f"{int((~torch.isfinite(got)).sum())} of {got.numel()} not finite"
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1, f"{worst:.3g} times the bound"


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("new,keys", [([152, 128, 72], [152, 128, 72]), ([4], [904])])
def test_hidden_values_of_the_largest_magnitude(dim, new, keys):
    """A hidden key's weight is zero, not merely small: 2^-126 of the type's largest value would be a number like 4. (The keys
    have the places 6 modulo 8.)"""
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = randn(g, sum(new), 4, dim), randn(g, sum(keys), 2, dim), randn(g, sum(keys), 2, dim)
    want, size = plain(q, k, v, new, keys)
    blind = torch.ones(sum(new), dtype=torch.bool, device=DEV)
    for s, (a, c, d) in enumerate(zip(offsets(new), offsets(keys), keys)):
        v[c + d - 2] = torch.finfo(torch.bfloat16).min if s % 2 else torch.finfo(torch.bfloat16).max
        blind[a + new[s] - 2:a + new[s]] = False  # the queries that see it
    got = packed(q, k, v, new, keys)
    check(got[blind], want[blind], size[blind])
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_scores_that_are_not_finite(dim, bad):
    """A key whose score is NaN or +inf, its value finite, at each of eight consecutive positions: queries that see it are
    NaN, the others and the other sequences know nothing of it."""
    g = torch.Generator(device=DEV).manual_seed(1)
    new = [150 + i for i in range(8)]
    n, off = sum(new), offsets(new)
    q, k, v = randn(g, n, 4, dim), randn(g, n, 2, dim), randn(g, n, 2, dim)
    q[:, :, 3] = 1.0
    want, size = plain(q, k, v, new, new)
    sees = torch.zeros(n, dtype=torch.bool, device=DEV)
    for s in range(8):
        at = off[s] + 64 + s
        k[at, :, 3] = bad
        sees[at:off[s + 1]] = True
    got = packed(q, k, v, new, new)
    assert bool(torch.isnan(got[sees]).all()), f"{int((~torch.isnan(got[sees])).sum())} results know nothing of the key"
    check(got[~sees], want[~sees], size[~sees])
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_scores_that_are_not_finite_in_cut_units(dim, bad):
    """The same where the units are cut along the keys."""
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = randn(g, 3, 2, dim), randn(g, 900, 2, dim), randn(g, 900, 2, dim)
    q[:, :, 3] = 1.0
    want, size = plain(q, k, v, [3], [900])
    for at in [*range(500, 508), 898]:
        kk = k.clone()
        kk[at, :, 3] = bad
        got = packed(q, kk, v, [3], [900])
        blind = 1 if at == 898 else 0  # query 0 does not see key 898
        assert bool(torch.isnan(got[blind:]).all()), f"key {at}"
        check(got[:blind], want[:blind], size[:blind]) if blind else None
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_a_part_whose_only_visible_key_is_nan(dim):
    """769 keys are seven tiles: the last part of a cut unit holds one key that the query sees."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = randn(g, 1, 1, dim), randn(g, 769, 1, dim), randn(g, 769, 1, dim)
    k[768] = NAN
    assert bool(torch.isnan(packed(q, k, v, [1], [769])).all())
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_cut_units_redo_the_dims_that_need_it(dim):
    """A hidden NaN in one dim of a cut unit's value: the blocks of 32 dims without it keep their bits, in every call."""
    g = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = randn(g, 40, 2, dim), randn(g, 5000, 2, dim), randn(g, 5000, 2, dim)
    want, size = plain(q, k, v, [40], [5000])
    clean = packed(q, k, v, [40], [5000])
    v[4998, :, 5] = NAN
    for _ in range(20):
        got = packed(q, k, v, [40], [5000])
        assert torch.equal(got[:38, :, 32:], clean[:38, :, 32:])
        check(got[:38], want[:38], size[:38])
        assert bool(torch.isnan(got[38:, :, 5]).all())
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_one_nan_value_that_most_queries_see(dim):
    """A NaN in one dim of an early value: NaN in that dim of the queries that see it, at a cost that does not grow with
    the keys of every query (each redone by itself over 30,000 keys took hundreds of milliseconds)."""
    g = torch.Generator(device=DEV).manual_seed(5)
    new, keys = [2048], [30000]
    q, k, v = randn(g, 2048, 8, dim), randn(g, 30000, 2, dim), randn(g, 30000, 2, dim)
    clean = packed(q, k, v, new, keys)
    v[7, 0, 5] = NAN
    v[20000, 1, 6] = INF
    got = packed(q, k, v, new, keys)
    torch.cuda.synchronize()
    start = time.perf_counter()
    got = packed(q, k, v, new, keys)
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    same = torch.ones_like(got, dtype=torch.bool)
    same[:, :4, 5] = False
    same[:, 4:, 6] = False
    assert torch.equal(got[same], clean[same])
    assert bool(torch.isnan(got[:, :4, 5]).all()) and bool((got[:, 4:, 6] == INF).all())
    assert kernels.read_status() == 0
    assert took < 0.1, f"{took:.3f} s"


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_values_whose_weighted_sum_overflows(dim):
    """Large values in a row whose running maximum lags behind its scores, so that the weights reach 2^7: the sum of the
    weighted values overflows, the result does not."""
    g = torch.Generator(device=DEV).manual_seed(6)
    n = 300
    q, k = randn(g, n, 2, dim), randn(g, n, 2, dim)
    k[:, :, 0] = torch.linspace(-2, 3, n, device=DEV)[:, None].to(torch.bfloat16)
    q[:, :, 0] = dim**0.5
    v = (randn(g, n, 2, dim).sign() * 2.0**118).to(torch.bfloat16)
    want, size = plain(q, k, v, [n], [n])
    check(packed(q, k, v, [n], [n]), want, size)
    assert kernels.read_status() == 0


def test_hidden_nan_after_many_keys():
    """The queries before a NaN value are redone from the formula, over as many keys as they see."""
    g = torch.Generator(device=DEV).manual_seed(7)
    new, keys = [200], [60000]
    q, k, v = randn(g, 200, 2, 128), randn(g, 60000, 1, 128), randn(g, 60000, 1, 128)
    want, size = plain(q, k, v, new, keys)
    v[59980] = NAN
    got = packed(q, k, v, new, keys)
    check(got[:180], want[:180], size[:180])
    assert bool(torch.isnan(got[180:]).all())
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_that_are_not_positive(dim, scale):
    """A scale of zero weighs all visible keys alike; a negative one prefers the smallest products."""
    g = torch.Generator(device=DEV).manual_seed(9)
    new, keys = [150, 40], [150, 300]
    q, k, v = randn(g, 190, 4, dim), randn(g, 450, 2, dim), randn(g, 450, 2, dim)
    want, size = plain(q, k, v, new, keys, scale)
    check(packed(q, k, v, new, keys, scale), want, size)
    assert kernels.read_status() == 0


@pytest.mark.parametrize("dim", [128, 512])
def test_rows_redone_for_longer_than_a_wait_may_last(dim):
    """127 queries over 260,000 keys do not see the last, NaN: their block redoes them for seconds, with a unit of a short
    sequence behind them, and no wait of the other warps gives up."""
    g = torch.Generator(device=DEV).manual_seed(11)
    n = 260000 if dim == 128 else 100000
    new, keys = [128] * 401, [n] + [128] * 400
    q, k, v = randn(g, sum(new), 1, dim), randn(g, sum(keys), 1, dim), randn(g, sum(keys), 1, dim)
    v[n - 1] = NAN
    got = packed(q, k, v, new, keys)
    assert kernels.read_status() == 0
    assert bool(torch.isnan(got[127]).all())
    v[n - 1] = 0.0
    want, size = plain(q, k, v, new, keys)
    rest = torch.arange(sum(new), device=DEV) != 127
    check(got[rest], want[rest], size[rest])


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 512)])
@pytest.mark.parametrize("tokens", [10, 5000])
def test_offsets_that_descend_are_reported(dtype, dim, tokens):
    q = torch.zeros(tokens, 2, dim, dtype=dtype, device=DEV)
    good = torch.tensor([0, 4, 4, tokens], device=DEV)
    kernels.packed_attention(q, q, q, good)
    assert kernels.read_status() == 0
    kernels.packed_attention(q, q, q, torch.tensor([0, 6, 4, tokens], device=DEV), good)
    assert kernels.read_status() == 1


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 128), (torch.bfloat16, 512)])
def test_strides_of_extents_of_one(dtype, dim):
    """The stride of an extent of one is not read, so it may be any number."""
    g = torch.Generator(device=DEV).manual_seed(10)
    q, k, v = (torch.randn(1, 1, dim, generator=g, device=DEV).to(dtype) for _ in range(3))
    odd = [torch.as_strided(t, t.shape, (3, 7, 1)) for t in (q, k, v)]
    off = torch.tensor([0, 1], device=DEV)
    assert torch.equal(kernels.packed_attention(*odd, off), v)
    pages = [torch.as_strided(t.view(1, 1, 1, dim), (1, 1, 1, dim), (5, 3, 1, 1)) for t in (k, v)]
    table, one = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int64, device=DEV)
    assert torch.equal(kernels.paged_attention(q, *pages, table, one, 0.1), v)
    kb, vb = kernels.paged_kv_read(*pages, table, off, 1)
    assert torch.equal(kb, k) and torch.equal(vb, v)
    cs = torch.zeros(1, dim // 2, 2, device=DEV)
    cs[..., 0] = 1
    qkv = torch.cat([q, k, v], -1).view(1, 3 * dim)
    fresh = [torch.zeros(1, 1, 1, dim, dtype=dtype, device=DEV) for _ in range(2)]
    into = [torch.as_strided(t, t.shape, (5, 3, 1, 1)) for t in fresh]
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    got = kernels.paged_rope_kv(torch.as_strided(qkv, qkv.shape, (1, 1)), cs, zero, *into, zero, 1, 1)
    assert torch.equal(got, q) and torch.equal(fresh[0].view(-1), k.view(-1)) and torch.equal(fresh[1].view(-1), v.view(-1))
    assert kernels.read_status() == 0
