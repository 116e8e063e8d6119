"""Attention over pages where the softmax is not an ordinary one.

Tolerances: see test_paged_gpu for the rounding of outputs, probabilities and sums."""

import time

import pytest
import torch

import paged_util as pu
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("heads,kv,dim,rows", [(8, 8, 128, 32), (16, 4, 128, 48), (16, 2, 64, 40), (32, 2, 128, 40), (8, 8, 512, 20), (8, 2, 256, 40)])
@pytest.mark.parametrize("n,nats", [*((32768, x) for x in (11.0, 11.4, 11.8, 12.2, 12.5, 13.0)), (131072, 13.0), (131072, 13.75)])
def test_a_key_far_above_a_long_tail(heads, kv, dim, rows, n, nats):
    """8-bit pages, one key 11 to 14 nats above the 32767 or 131071 others that score alike, values with a common mean: each
    weight of the tail lies around or below the smallest step of the two e4m3 pieces (2^-13; the key's weight is 2^4 to
    2^8), yet together they are 7 to 35% of the sum. The units are long enough that few are cut.

    Beside the rounding of the output and of the weights' 8 significant bits (2^-8 (|o| + A), 2^-10 A), a weight's last piece
    is off by an error of mean zero within one step, a standard deviation of at most half of one: over n keys and a sum l >= 2^4
    that is sqrt(n) 2^-14 / l of a value; six of them (2.4e5 results, about 5e-4 of one expected past it)."""
    page = 128
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.zeros(n // page, kv, page, dim, device=DEV)
    k[3, :, 77, 0] = 1.0
    v = 1.0 + 0.25 * torch.randn(n // page, kv, page, dim, generator=g, device=DEV)
    v[3, :, 77] = -1.0
    k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    ones = torch.full(k.shape[:3], 127, dtype=torch.uint8, device=DEV)
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).expand(rows, -1).contiguous()
    q = torch.zeros(rows, heads, dim, device=DEV, dtype=torch.bfloat16)
    q[:, :, 0] = nats
    got = kernels.paged_attention(q, k, v, table, torch.full((rows,), n, device=DEV), 1.0, k_scale=ones, v_scale=ones).double()
    x = torch.zeros(n, dtype=torch.float64, device=DEV)
    x[3 * page + 77] = float(q[0, 0, 0])
    p = torch.softmax(x, 0)
    want = torch.einsum("j,hjd->hd", p, v.double().transpose(0, 1).reshape(kv, n, dim)).repeat_interleave(heads // kv, 0)
    size = torch.einsum("j,hjd->hd", p, v.double().abs().transpose(0, 1).reshape(kv, n, dim)).repeat_interleave(heads // kv, 0)
    noise = 6 * n**0.5 * 2.0**-14 / 2.0**4 * float(v.double().abs().max())
    bound = 2.0**-8 * (want.abs() + size) + 2.0**-10 * size + noise
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1, f"{worst:.3g} times the bound"
    assert kernels.read_status() == 0


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (2, 2, 512), (4, 2, 256)])
def test_one_nan_value_that_all_drafts_see(kind, heads, kv, dim):
    """A NaN in one dim of an early value of long rows, five draft tokens: NaN in that dim, the other dims as without it, and
    no column walks its 60,000 keys one after the other for it (which took tens of milliseconds)."""
    g = torch.Generator(device=DEV).manual_seed(3)
    n, page, t, rows = 60000, 32, 5, 4
    k, v = (torch.randn(n // page, kv, page, dim, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    ones = None
    if kind == "fp8":
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ones = torch.full(k.shape[:3], 127, dtype=torch.uint8, device=DEV)
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).expand(rows, -1).contiguous()
    q = torch.randn(rows * t, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    run = lambda: kernels.paged_attention(q, k, v, table, torch.full((rows,), n - t + 1, device=DEV), dim**-0.5, tokens=t,  # noqa: E731
                                          k_scale=ones, v_scale=ones)
    clean = run()
    v.view(torch.uint8 if kind == "fp8" else v.dtype)[0, :, 7, 5] = 0x7F if kind == "fp8" else NAN
    run()
    torch.cuda.synchronize()
    start = time.perf_counter()
    got = run()
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    same = torch.arange(dim, device=DEV) != 5
    assert torch.equal(got[..., same], clean[..., same])
    assert bool(torch.isnan(got[..., 5]).all())
    assert kernels.read_status() == 0
    assert took < 5e-3, f"{took:.4f} s"


@pytest.mark.parametrize("kind", ["own", "fp8"])
def test_drafts_after_many_keys_leave_a_hidden_nan_out(kind):
    """The draft columns before a NaN are redone over all their keys."""
    g = torch.Generator(device=DEV).manual_seed(4)
    n, page, t, kv, dim = 60000, 32, 5, 2, 128
    k, v = (torch.randn(n // page, kv, page, dim, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    ones = None
    if kind == "fp8":
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ones = torch.full(k.shape[:3], 127, dtype=torch.uint8, device=DEV)
    kk, vv = (x.double().transpose(0, 1).reshape(kv, n, dim) for x in (k, v))
    table = torch.arange(n // page, dtype=torch.int32, device=DEV)[None]
    q = torch.randn(t, 4, dim, generator=g, device=DEV).to(torch.bfloat16)
    v.view(torch.uint8 if kind == "fp8" else v.dtype)[-1, :, page - 2] = 0x7F if kind == "fp8" else NAN  # key n - 2
    got = kernels.paged_attention(q, k, v, table, torch.full((1,), n - t + 1, device=DEV), dim**-0.5, tokens=t, k_scale=ones,
                                  v_scale=ones).double()
    for i in range(t - 2):
        m = n - t + 1 + i
        p = torch.softmax(q[i].double().view(kv, 2, dim) @ kk[:, :m].transpose(1, 2) * dim**-0.5, -1)
        want, size = ((p @ x[:, :m]).view(4, dim) for x in (vv, vv.abs()))
        assert float(((got[i] - want).abs() / (2.0**-8 * (want.abs() + size) + 2.0**-10 * size)).max()) <= 1
    assert bool(torch.isnan(got[t - 2:]).all())
    assert kernels.read_status() == 0


@pytest.mark.parametrize("kind", ["own", "fp8"])
def test_columns_redone_for_longer_than_a_wait_may_last(kind):
    """Draft columns over a million and a half keys (a few pages, over and over) with a hidden NaN behind them, and short rows
    after them: the redo takes seconds, and no wait gives up."""
    g = torch.Generator(device=DEV).manual_seed(5)
    page, t, kv, dim, real, width, short = 64, 5, 1, 128, 8, 24000, 300
    k, v = (torch.randn(real + 1, kv, page, dim, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    ones = None
    if kind == "fp8":
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ones = torch.full(k.shape[:3], 127, dtype=torch.uint8, device=DEV)
    table = (torch.arange(width, dtype=torch.int32, device=DEV) % real).expand(1 + short, -1).contiguous()
    table[0, width - 1] = real
    n = width * page
    lengths = torch.full((1 + short,), 3 * page, device=DEV)
    lengths[0] = n - t + 1
    kk, vv = (torch.cat([x[i % real] if i < width - 1 else x[real] for i in range(width - 2 * real, width)], 1).double() for x in (k, v))
    copies = torch.ones(kk.size(1), dtype=torch.float64, device=DEV)  # of each of these keys in the row
    copies[:real * page] += width // real - 2
    q = torch.randn((1 + short) * t, 4, dim, generator=g, device=DEV).to(torch.bfloat16)
    v.view(torch.uint8 if kind == "fp8" else v.dtype)[real, :, page - 1] = 0x7F if kind == "fp8" else NAN
    got = kernels.paged_attention(q, k, v, table, lengths, dim**-0.5, tokens=t, k_scale=ones, v_scale=ones).double()
    assert kernels.read_status() == 0
    assert bool(torch.isnan(got[t - 1]).all()) and bool(torch.isfinite(got[t:]).all())
    for i in range(t - 1):
        m = kk.size(1) - t + 1 + i
        x = q[i].double() @ kk[0, :m].t() * dim**-0.5 + copies[:m].log()
        p = torch.softmax(x, -1)
        want, size = p @ vv[0, :m], p @ vv[0, :m].abs()
        # (fp32 sums over 1.5 million keys one after the other: 2^-24 of the sum each, in a direction that wanders)
        assert float(((got[i] - want).abs() / (2.0**-8 * (want.abs() + size) + 2.0**-10 * size)).max()) <= 1


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 128, 16), (16, 1, 128, 64), (4, 4, 512, 64), (8, 1, 64, 16), (4, 1, 256, 128)])
def test_minus_infinity_before_scores_far_below_zero(heads, kv, dim, page):
    """The first 256 keys score -inf, the later ones about -250: a column's maximum starts at the first score that is one. (The
    rows are short enough to stay whole: each softmax group meets -inf alone in its first tile.)"""
    g = torch.Generator().manual_seed(2)
    lens = [600, 300, 520]
    table, pool = pu.table_for(lens, page, g)
    k, v, _, _, _, _ = pu.cache(pool, kv, page, dim, "own", g)
    q = torch.randn(len(lens), heads, dim, generator=g).to(torch.bfloat16)
    q[:, :, 3], q[:, :, 4] = 1.0, 16.0
    for r, n in enumerate(lens):
        for j in range(n):
            k[int(table[r, j // page]), :, j % page, 4] = -16.0
            if j < 256:
                k[int(table[r, j // page]), :, j % page, 3] = -INF
    length = torch.tensor(lens)
    want = pu.paged(q, k, v, table, length, 1.0, 1)
    size = pu.paged(q, k, v.abs(), table, length, 1.0, 1)
    got = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), length.to(DEV), 1.0).double().cpu()
    # (fp32 scores of about 370 in log2 units: a relative 2^-24 of them is 2^-15 of a weight)
    bound = 2.0**-8 * (want.abs() + size) + 2.0**-10 * size
    worst = float(((got - want).abs() / bound).nan_to_num(INF).max())
    assert worst <= 1, f"{worst:.3g} times the bound"
    assert kernels.read_status() == 0


def test_rows_of_two_billion_keys():
    """A table of one page 16.8 million times over: keys up to the largest that a row may have, and lengths past it, which are
    reported and stay within the table."""
    g = torch.Generator(device=DEV).manual_seed(6)
    page, dim, t = 128, 64, 2
    width = 0x7fffff00 // page
    k, v = (torch.randn(1, 1, page, dim, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(t, 2, dim, generator=g, device=DEV).to(torch.bfloat16)
    table = torch.zeros(1, width, dtype=torch.int32, device=DEV)
    run = lambda n: kernels.paged_attention(q, k, v, table, torch.tensor([n], device=DEV), dim**-0.5, tokens=t).double()  # noqa: E731
    got = run(width * page - 1)
    assert kernels.read_status() == 0
    p = torch.softmax(q.double() @ k[0, 0].double().t() * dim**-0.5, -1)
    want, size = p @ v[0, 0].double(), p @ v[0, 0].double().abs()
    # Beside the usual rounding, sums of 57,000 tiles per block, each added to 2^-24 of the sum at most: 57000 x 2^-24 < 2^-8.
    assert float(((got - want).abs() / (2.0**-8 * (want.abs() + 2 * size) + 2.0**-10 * size)).max()) <= 1
    for n in (width * page, 2**31 - 1, 2**31, 2**40, 2**63 - 1):
        run(n)
        assert kernels.read_status() == 1


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 16), (torch.float32, 64, 16), (torch.bfloat16, 32, 5)])
def test_lengths_at_the_ends_of_their_type(dtype, dim, page):
    g = torch.Generator(device=DEV).manual_seed(7)
    k, v = (torch.randn(3, 1, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(6, 2, dim, generator=g, device=DEV).to(dtype)
    table = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    good = kernels.paged_attention(q, k, v, table, torch.tensor([3, 4, 2], device=DEV), 0.1, tokens=2)
    assert kernels.read_status() == 0
    for n in (2**63 - 1, -2**63):
        out = kernels.paged_attention(q, k, v, table, torch.tensor([3, n, 2], device=DEV), 0.1, tokens=2)
        assert kernels.read_status() == 1
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])
