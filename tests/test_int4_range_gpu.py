"""Attention over 4-bit pages whose values' scales differ widely: between keys, between the groups of 32 dims of a vector, between blocks
of keys, and as a whole; against float64.

The bound of test_int4_cache_gpu.py, 2^-8 |o| + (2^-11 + 2^-10) A + 2^-11 B with A = sum p |v| / sum p and B = sum p |s| / sum p, and what
fp16 loses below its normal numbers. A weight is 2^12 or more where it is a warp's largest, and a scale that fp16 sees is taken relative to a
power of two that is at most 2^11 times it; so half a step of fp16's smallest numbers, 2^-25, is at most 2^-25 2^-12 2^11 = 2^-26 of the
largest weight times the key's scale, and times a code of at most 8 2^-23 of it. Keys whose scales lie further apart than 2^13 within
their 16 are summed in fp32, so a scale counts for at most 2^13 times the least (of those that are not 0) among its key's 16:
2^-23 C with C = max p * sum min(|s|, 2^13 least) / sum p."""

import pytest
import torch

import int4_util as iu
import paged_util as pu
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
dev = lambda t: t.to(DEV)  # noqa: E731


def want_of(q, kval, vval, vs, table, lens, scale, tokens, page):
    """(o, bound) in float64, row by row."""
    heads, kv, dim = q.size(1), kval.size(1), kval.size(3)
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for r, n in enumerate(lens):
        most = n + tokens - 1
        if most <= 0:
            continue
        ids = table[r, : -(-most // page)].long()
        rows = lambda t: t[ids].double().transpose(1, 2).reshape(-1, kv, t.size(3))[:most]  # noqa: E731
        k, v, s = rows(kval), rows(vval), rows(vs.float().abs())
        pad = torch.full((-most % 16, kv, s.size(2)), float("inf"), dtype=torch.float64)
        least = torch.cat([torch.where(s == 0, float("inf"), s), pad]).unflatten(0, (-1, 16)).amin(1)
        least = torch.where(least.isinf(), 0.0, least).repeat_interleave(16, 0)[:most]
        held = torch.minimum(s, 2.0**13 * least)
        for t in range(tokens):
            m = n + t
            if m <= 0:
                continue
            for h in range(heads):
                j = h * kv // heads
                p = torch.softmax(k[:m, j] @ q[r * tokens + t, h].double() * scale, 0)
                o = p @ v[:m, j]
                wide = lambda x: x.repeat_interleave(32, -1)  # noqa: E731
                a, b, c = p @ v[:m, j].abs(), wide(p @ s[:m, j]), wide(p.max() * held[:m, j].sum(0))
                out[r * tokens + t, h] = o
                bound[r * tokens + t, h] = 2.0**-8 * o.abs() + (2.0**-11 + 2.0**-10) * a + 2.0**-11 * b + 2.0**-23 * c + 2.0**-133
    return out, bound


def run(heads, kv, dim, page, lens, tokens, sizes, seed, low=(), rising=0.0, scale=None, wide=False):
    """`sizes(exponent [keys, groups], g)` sets the power of two of each position's groups of V in row order; the keys `low` get scores
    far below the others'; `rising`: how much the scores grow over a row; `wide`: tables with room for so many keys that a unit takes
    all the columns it can."""
    g = torch.Generator().manual_seed(seed)
    covered = [max(0, n + tokens - 1) for n in lens]
    table, pool = pu.table_for(covered, page, g, 2)
    base = torch.randn(kv, dim, generator=g)
    x = {True: torch.randn(pool, kv, page, dim, generator=g), False: torch.randn(pool, kv, page, dim, generator=g)}
    for r, n in enumerate(covered):
        e = torch.zeros(n, dim // 32, dtype=torch.int64)
        sizes(e, g)
        for j in range(n):
            at = int(table[r, j // page]), slice(None), j % page
            x[False][at] *= torch.pow(2.0, e[j].double()).repeat_interleave(32).float()
            if j in low:
                x[True][at] = -4 * base
            elif rising:
                x[True][at] = 0.3 * x[True][at] + base * (rising * j / n)
    stored = []
    for keys in (True, False):
        codes, s = iu.quantise(x[keys].bfloat16())
        stored.append((iu.pack(codes, keys), s, iu.values(codes, s)))
    (k, ks, kval), (v, vs, vval) = stored
    q = (base.repeat_interleave(heads // kv, 0) + 0.3 * torch.randn(len(lens) * tokens, heads, dim, generator=g)).bfloat16()
    scale = dim**-0.5 if scale is None else scale
    want, bound = want_of(q, kval, vval, vs, table, lens, scale, tokens, page)
    if wide:
        table = torch.cat([table, torch.zeros(len(lens), 100_000 // page, dtype=torch.int32)], 1)
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), torch.tensor(lens, device=DEV), scale, tokens=tokens,
                                  k_scale=dev(ks), v_scale=dev(vs)).double().cpu()
    assert bool(torch.isfinite(got).all()), "not finite"
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} past the bound; worst {float(((got - want).abs() / bound).max()):.3g} times"
    assert kernels.read_status() == 0


SHAPES = [(4, 4, 64, 16, 1), (12, 2, 64, 32, 3), (16, 1, 64, 128, 2), (4, 4, 128, 64, 1), (8, 2, 128, 16, 5), (12, 1, 128, 12, 2), (32, 1, 128, 32, 1),
          (4, 2, 256, 16, 1), (16, 1, 256, 64, 1), (2, 2, 512, 64, 1), (8, 1, 512, 8, 2)]
LENS = [1, 15, 40, 130, 700]


@pytest.mark.parametrize("by", [10, 14, 20, 26, 30, 40])
@pytest.mark.parametrize("heads,kv,dim,page,tokens", SHAPES)
def test_a_key_of_little_weight_with_large_values(heads, kv, dim, page, tokens, by):
    """Keys of every warp's first blocks whose values are 2^by times the others' and whose weights are next to nothing."""
    places = (0, 3, 17, 40, 75, 101, 127, 333)

    def sizes(e, g):
        for j in places:
            if j < len(e):
                e[j] += by

    run(heads, kv, dim, page, LENS, tokens, sizes, by + dim, low=places)


@pytest.mark.parametrize("by", [8, 24, 40])
@pytest.mark.parametrize("heads,kv,dim,page,tokens", SHAPES)
def test_a_key_whose_values_make_up_for_its_weight(heads, kv, dim, page, tokens, by):
    run(heads, kv, dim, page, LENS, tokens, lambda e, g: e[5::50].add_(by), by * dim)


@pytest.mark.parametrize("heads,kv,dim,page,tokens", SHAPES)
def test_groups_of_different_size(heads, kv, dim, page, tokens):
    """The groups of one vector 2^20 and more apart, the same in every key."""
    sizes = torch.tensor([0, -20, 20, -36, 3, 30, -12, 8] * 2)
    run(heads, kv, dim, page, LENS, tokens, lambda e, g: e.add_(sizes[: e.size(1)]), dim)


@pytest.mark.parametrize("most", [4, 12, 30])
@pytest.mark.parametrize("heads,kv,dim,page,tokens", SHAPES)
def test_groups_of_random_size(heads, kv, dim, page, tokens, most):
    """Every group of every key with a size of its own."""
    run(heads, kv, dim, page, LENS, tokens, lambda e, g: e.add_(torch.randint(-most, most + 1, e.shape, generator=g)), dim + most)


@pytest.mark.parametrize("rising", [0.0, 3.0])
@pytest.mark.parametrize("heads,kv,dim,page,tokens", SHAPES)
def test_blocks_of_different_size(heads, kv, dim, page, tokens, rising):
    """Runs of keys whose sizes go up and down by 2^30; with scores that grow, so that sums are scaled down meanwhile."""
    def sizes(e, g):
        for i in range(0, len(e), 16):
            e[i:i + 16] += [0, 30, 30, -10, 0, 0, -30, 5][i // 32 % 8]

    run(heads, kv, dim, page, LENS, tokens, sizes, dim, rising=rising)


@pytest.mark.parametrize("all_by", [-110, -70, 70, 100])
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_values_all_tiny_or_huge(dim, all_by):
    run(4, 2, dim, 16, LENS, 2, lambda e, g: e.add_(all_by + torch.randint(-1, 2, e.shape, generator=g)), dim)


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_groups_that_are_zero(dim):
    """A group that is zero in every key, one that is in every other, one that is in whole blocks."""
    def sizes(e, g):
        e[:, 0] = -2000
        e[::2, 1] = -2000
        if e.size(1) > 2:
            e[64:200, 2] = -2000

    run(4, 2, dim, 16, LENS, 1, sizes, dim)


@pytest.mark.parametrize("dim", [64, 128, 512])
def test_drafts_do_not_spoil_the_queries_before_them(dim):
    """The last drafts' values are 2^40 times the cache's: the queries that do not see them keep their bound."""
    def sizes(e, g):
        e[-2:] += 40

    run(8, 2, dim, 16, [5, 30, 64, 200], 4, sizes, dim)


# heads, kv heads, tokens whose columns make 2, 3, 4 and 2 x 3 tiles of 8 (256 dims: 2 and 2 x 2)
COLUMNS = [(32, 8, 4), (32, 8, 5), (16, 1, 2), (40, 1, 1), (7, 1, 2)]


@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,tokens", COLUMNS)
def test_units_of_several_tiles(heads, kv, tokens, dim, page):
    """Tame values, groups and keys of every size, and scores that grow, with all of a unit's columns at once."""
    lens = [0, 3, 33, 64, 300]
    args = (heads, kv, dim, page, lens, tokens)
    run(*args, lambda e, g: None, dim, wide=True)
    run(*args, lambda e, g: e.add_(torch.randint(-12, 13, e.shape, generator=g)), dim + 1, wide=True)
    run(*args, lambda e, g: e[5::50].add_(24), dim + 2, wide=True, rising=2.0)


@pytest.mark.parametrize("heads,kv,dim,page,n,tokens", [(32, 8, 128, 64, 4000, 5), (16, 2, 64, 16, 4500, 3), (16, 1, 256, 32, 3000, 2), (40, 1, 128, 16, 4900, 2)])
def test_long_rows_in_several_tiles(heads, kv, dim, page, n, tokens):
    """Units that are cut between many CTAs, of several tiles of columns, with keys and groups of different sizes."""
    run(heads, kv, dim, page, [n, n // 3], tokens, lambda e, g: e.add_(torch.randint(-6, 7, (len(e) // 64 + 1, e.size(1)), generator=g)
                                                                      .repeat_interleave(64, 0)[: len(e)]), n, wide=True)
