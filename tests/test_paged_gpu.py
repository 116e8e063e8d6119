"""The paged cache (write, read back, attention) and the packed-prompt attention on the GPU, against the plain forms in 64
bits of paged_util.

Tolerances. fp32: 2e-5 (1 + |o|), the framework's own for fp32 attention. bf16: the output's rounding is at most 2^-8 |o|;
the probabilities enter the second product in 8 significant bits (bf16, or two e4m3 pieces), at most 2^-8 of each, which
moves o by at most 2^-8 A with A = sum p |v| / sum p; with e4m3 pieces also by half of their smallest step, 2^-18 of the
largest probability and key; fp32 sums and the exponential add well under 2^-10 A. Writes and read-backs are exact."""

import pytest
import torch

import paged_util as pu
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def check(got, want, size, dtype, fp8_keys=0, vmax=0.0):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), "not finite"
    if dtype == torch.float32:
        bound = 2e-5 * (1 + want.abs())
    else:
        bound = 2.0**-8 * (want.abs() + size) + 2.0**-10 * size + fp8_keys * 2.0**-18 * vmax + 1e-30
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} past the bound; worst " \
                                f"{float(((got - want).abs() / bound).max()):.3g} times"
    assert kernels.read_status() == 0


def spoil(k, v, ks, vs, table, lens, page):
    """NaN into every position of the pages that no row's length covers (pages of no row included)."""
    used = torch.zeros(k.size(0), page, dtype=torch.bool)
    for r, n in enumerate(lens):
        for j in range(n):
            used[int(table[r, j // page]), j % page] = True
    for t in (k, v):
        raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        raw.permute(0, 2, 1, 3)[~used] = 0x7F if t.dtype == torch.float8_e4m3fn else float("nan")
    for t in (ks, vs):
        if t is not None:
            t.permute(0, 2, 1)[~used] = 200


def run_paged(heads, kv, dim, page, lens, tokens, dtype, kind, seed=0, layout="page", spare=2):
    g = torch.Generator().manual_seed(seed)
    covered = [max(0, n + tokens - 1) for n in lens]
    table, pool = pu.table_for(covered, page, g, spare)
    k, v, ks, vs, kval, vval = pu.cache(pool, kv, page, dim, kind, g, DT[dtype])
    q = torch.randn(len(lens) * tokens, heads, dim, generator=g).to(DT[dtype])
    scale = dim**-0.5
    length = torch.tensor(lens)
    want = pu.paged(q, kval, vval, table, length, scale, tokens)
    size = pu.paged(q, kval, vval.abs(), table, length, scale, tokens)
    spoil(k, v, ks, vs, table, covered, page)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    k, v = dev(k), dev(v)
    if layout == "token":  # [pages, page, kv, D] storage
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif layout == "both":  # K and V of a page side by side
        kvp = torch.stack([k.view(torch.uint8) if kind == "fp8" else k, v.view(torch.uint8) if kind == "fp8" else v], 1)
        k, v = (kvp[:, i].view(k.dtype) for i in range(2))
    got = kernels.paged_attention(dev(q), k, v, dev(table), dev(length), scale, tokens=tokens, k_scale=dev(ks), v_scale=dev(vs))
    check(got, want, size, DT[dtype], max(covered) if kind == "fp8" else 0, float(vval.abs().max()))
    again = kernels.paged_attention(dev(q), k, v, dev(table), dev(length), scale, tokens=tokens, k_scale=dev(ks), v_scale=dev(vs))
    assert torch.equal(got, again), "two calls differ"


LENS = [0, 1, 2, 15, 16, 17, 127, 128, 129, 300, 511, 700]


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim,page,dtype", [
    (8, 2, 128, 16, "bf16"), (4, 4, 128, 64, "bf16"), (6, 2, 128, 8, "bf16"), (32, 1, 128, 32, "bf16"), (16, 1, 128, 128, "bf16"),
    (4, 4, 512, 64, "bf16"), (8, 1, 512, 16, "bf16"), (4, 2, 256, 16, "bf16"), (3, 3, 64, 16, "bf16"), (4, 1, 128, 12, "bf16"),
    (4, 2, 128, 256, "bf16"), (2, 2, 32, 4, "bf16"), (2, 1, 16, 1, "bf16"), (8, 2, 64, 32, "bf16"), (16, 1, 64, 128, "bf16"), (20, 1, 256, 64, "bf16"),
    (4, 2, 64, 16, "f32"), (3, 1, 128, 16, "f32"), (2, 2, 512, 8, "f32"), (4, 4, 16, 5, "f32"), (8, 1, 256, 16, "f32")])
def test_paged_one_token(heads, kv, dim, page, dtype, kind):
    run_paged(heads, kv, dim, page, LENS, 1, dtype, kind)


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim,page,tokens,dtype", [
    (4, 4, 128, 64, 5, "bf16"), (8, 2, 128, 16, 2, "bf16"), (8, 2, 128, 16, 4, "bf16"), (8, 2, 128, 16, 7, "bf16"), (8, 2, 64, 16, 5, "bf16"), (4, 2, 256, 16, 3, "bf16"),
    (2, 2, 512, 32, 8, "bf16"), (4, 2, 64, 16, 3, "f32"), (6, 2, 128, 16, 1, "bf16"), (10, 2, 128, 32, 3, "bf16")])
def test_paged_drafts(heads, kv, dim, page, tokens, dtype, kind):
    run_paged(heads, kv, dim, page, [0, 1, 3, 16, 120, 126, 127, 128, 130, 385], tokens, dtype, kind, seed=3)


@pytest.mark.parametrize("layout", ["token", "both"])
@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "bf16"), (512, "bf16"), (64, "f32")])
def test_paged_other_layouts(layout, kind, dim, dtype):
    run_paged(4, 2, dim, 16, [5, 40, 260], 1, dtype, kind, seed=4, layout=layout)


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (2, 2, 512)])
def test_paged_long_row(kind, heads, kv, dim):
    """One row over most of the GPU's CTAs: its splits are joined."""
    run_paged(heads, kv, dim, 32, [5003], 1, "bf16", kind, seed=5)


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim,page,rows,n", [(8, 4, 128, 8, 40, 3000), (4, 4, 512, 16, 20, 1500), (4, 2, 256, 64, 40, 2500),
                                                      (32, 2, 64, 32, 60, 2000), (32, 2, 128, 128, 40, 2500), (16, 1, 512, 32, 30, 2000)])
def test_paged_batches(kind, heads, kv, dim, page, rows, n):
    """Ragged batches that send every CTA through many tiles and several segments (ring slots that hold K and V in turn),
    against the formula in float64 on the GPU."""
    g = torch.Generator().manual_seed(rows)
    lens = [n - (i * 977) % n for i in range(rows)]
    table, pool = pu.table_for(lens, page, g)
    cg = torch.Generator(device=DEV).manual_seed(1)
    pages, scales, values = [], [], []
    for _ in range(2):
        x = torch.randn(pool, kv, page, dim, generator=cg, device=DEV).to(torch.bfloat16)
        if kind == "fp8":
            e = torch.frexp(x.float().abs().amax(-1))[1] - 8  # (any exponent that holds the vector)
            codes = torch.ldexp(x.float(), -e[..., None]).to(torch.float8_e4m3fn)
            pages.append(codes)
            scales.append((e + 127).to(torch.uint8))
            values.append(codes.float() * 2.0 ** e.float()[..., None])
        else:
            pages.append(x)
            scales.append(None)
            values.append(x)
    q = torch.randn(rows, heads, dim, generator=cg, device=DEV).to(torch.bfloat16)
    got = kernels.paged_attention(q, *pages, table.to(DEV), torch.tensor(lens, device=DEV), dim**-0.5, k_scale=scales[0],
                                  v_scale=scales[1])
    for r, m in enumerate(lens):
        ids = table[r].long().to(DEV)[: -(-m // page)]
        k, v = (t[ids].double().transpose(0, 1).reshape(kv, -1, dim)[:, :m] for t in values)
        qr = q[r].double().view(kv, heads // kv, dim)
        p = torch.softmax(qr @ k.transpose(1, 2) * dim**-0.5, -1)
        want, size = ((p @ t).view(heads, dim).cpu() for t in (v, v.abs()))
        check(got[r], want, size, torch.bfloat16, m if kind == "fp8" else 0, float(v.abs().max()))


@pytest.mark.parametrize("kind", ["own", "fp8"])
def test_paged_many_rows(kind):
    """More rows than one launch schedules at a time, most of them short, many empty."""
    run_paged(2, 2, 128, 16, [(i * 37) % 50 for i in range(1500)], 1, "bf16", kind, seed=6)


@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (512, "bf16"), (32, "f32")])
def test_paged_scores_far_apart(kind, dim, dtype):
    """Scores that grow by hundreds along the keys, and a first key far below: the running maximum has to follow; values
    whose scales differ by 2^40."""
    g = torch.Generator().manual_seed(7)
    lens, page = [700, 129], 16
    table, pool = pu.table_for(lens, page, g)
    k, v, ks, vs, kval, vval = pu.cache(pool, 1, page, dim, "own", g, DT[dtype])
    flat = [int(table[0, j // page]) * page + j % page for j in range(700)]
    kk = k.permute(0, 2, 1, 3).reshape(-1, dim)
    for j, at in enumerate(flat):
        kk[at] = 0.05 * torch.randn(dim, generator=g)
        kk[at, 0] = (j - 400) * 0.5 if j < 600 else -300.0
    vv = v.permute(0, 2, 1, 3).reshape(-1, dim)
    vv[flat[598]] *= 2.0**-20
    vv[flat[599]] *= 2.0**20
    k, v = (t.view(pool, page, 1, dim).permute(0, 2, 1, 3).contiguous() for t in (kk, vv))
    if kind == "fp8":
        (k, ke), (v, ve) = pu.quantise(k), pu.quantise(v)
        ks, vs = (ke + 127).to(torch.uint8), (ve + 127).to(torch.uint8)
        kval, vval = pu.dequantise(k, ks), pu.dequantise(v, vs)
    else:
        kval, vval = k, v
    q = torch.zeros(2, 2, dim)
    q[:, 0, 0], q[:, 1, 0] = 3.0, -2.0
    q = (q + 0.1 * torch.randn(2, 2, dim, generator=g)).to(DT[dtype])
    length = torch.tensor(lens)
    want = pu.paged(q, kval, vval, table, length, 1.0, 1)
    size = pu.paged(q, kval, vval.abs(), table, length, 1.0, 1)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(length), 1.0, k_scale=dev(ks), v_scale=dev(vs))
    if dtype == "f32":  # scores of about 300 in fp32: a relative 2^-24 of them is 2e-5 of a probability
        assert bool(((got.double().cpu() - want).abs() <= 2e-4 * (size + 1e-30)).all())
    else:
        check(got, want, size * 1.01, DT[dtype], 0, 0)


def test_paged_nan_of_a_later_draft_token_stays_out():
    """A draft token's value that is NaN reaches the queries that see it and no other."""
    g = torch.Generator().manual_seed(8)
    t, page, n = 3, 16, 40
    table, pool = pu.table_for([n + t - 1], page, g)
    k, v, _, _, _, _ = pu.cache(pool, 2, page, 128, "own", g)
    want_v = v.clone()
    last = n + t - 2
    v[int(table[0, last // page]), :, last % page] = float("nan")
    k[int(table[0, last // page]), :, last % page] = float("nan")
    q = torch.randn(t, 4, 128, generator=g).to(torch.bfloat16)
    length = torch.tensor([n])
    want = pu.paged(q, k, want_v, table, length, 0.1, t)
    got = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), length.to(DEV), 0.1, tokens=t).cpu()
    assert bool(torch.isnan(got[2]).all())
    assert bool(torch.isfinite(got[:2]).all())
    assert float((got[:2].double() - want[:2]).abs().max()) <= 2e-2


def test_paged_bad_pages_and_lengths_are_reported():
    g = torch.Generator().manual_seed(9)
    k, v, _, _, _, _ = pu.cache(6, 2, 16, 128, "own", g)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    q = torch.randn(2, 4, 128, generator=g).to(torch.bfloat16)
    length = torch.tensor([40, 33])
    good = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), length.to(DEV), 0.1)
    assert kernels.read_status() == 0
    for bad in (-1, 6, 2**31 - 1):
        t = table.clone()
        t[0, 1] = bad
        out = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), t.to(DEV), length.to(DEV), 0.1)
        assert kernels.read_status() == 1
        assert torch.equal(out[1], good[1])
    for n in (-3, 49, 2**40):
        out = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor([n, 33]).to(DEV), 0.1)
        assert kernels.read_status() == 1
        assert torch.equal(out[1], good[1])


# ---------------------------------------------------------------------------------------------------------------- cache

@pytest.mark.parametrize("kind", ["own", "fp8"])
@pytest.mark.parametrize("heads,kv,dim,page,n,dtype", [
    (8, 2, 128, 16, 1, "bf16"), (8, 2, 128, 16, 37, "bf16"), (32, 8, 128, 64, 300, "bf16"), (8, 8, 512, 64, 19, "bf16"),
    (3, 1, 256, 8, 11, "bf16"), (5, 5, 64, 16, 23, "bf16"), (2, 1, 32, 3, 9, "bf16"), (2, 2, 16, 1, 5, "bf16"),
    (4, 2, 128, 16, 21, "f32"), (2, 2, 512, 16, 6, "f32"), (4, 1, 16, 7, 13, "f32"), (33, 3, 64, 16, 2, "f32")])
def test_write_and_read_back(heads, kv, dim, page, n, dtype, kind):
    """Bit-exact: q, the pages' codes and scale bytes, nothing else written, and the read-back."""
    g = torch.Generator().manual_seed(n * 7 + dim)
    pool = -(-n // page) + 4
    k, v, ks, vs, _, _ = pu.cache(pool, kv, page, dim, kind, g, DT[dtype])
    x = torch.randn(n, heads + 2 * kv, dim, generator=g) * torch.exp(3 * torch.randn(n, heads + 2 * kv, 1, generator=g))
    x[0, heads] = 0.0
    if n > 4:
        x[3, heads + kv] *= 2.0**-70  # scales held at their ends
        x[4, heads + kv] *= 2.0**60
    x = x.to(DT[dtype])
    pos = torch.randint(0, 900, (n,), generator=g)
    ang = torch.rand(900, dim // 2, generator=g, dtype=torch.float64) * 6.28
    cs = torch.stack([ang.cos(), ang.sin()], -1).float()
    slots = torch.randperm(pool * page, generator=g)[:n]
    if n > 8:
        slots[7] = -1
    turned = pu.rope(x[:, : heads + kv], cs[pos])
    keep = slots >= 0
    want = [k.clone(), v.clone()]
    want_s = [None if t is None else t.clone() for t in (ks, vs)]
    for i, r in enumerate((turned[:, heads:], x[:, heads + kv:])):
        at, off = slots[keep] // page, slots[keep] % page
        if kind == "fp8":
            codes, e = pu.quantise(r[keep])
            want[i].view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            want_s[i][at, :, off] = (e + 127).to(torch.uint8)
        else:
            want[i][at, :, off] = r[keep]
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    kd, vd, ksd, vsd = dev(k), dev(v), dev(ks), dev(vs)
    wide = torch.zeros(n, x[0].numel() + 32, dtype=x.dtype, device=DEV)  # rows further apart than they are long
    wide[:, : x[0].numel()] = dev(x.reshape(n, -1))
    q = kernels.paged_rope_kv(wide[:, : x[0].numel()], dev(cs), dev(pos), kd, vd, dev(slots), heads, kv, k_scale=ksd, v_scale=vsd)
    assert torch.equal(q.cpu(), turned[:, :heads])
    raw = lambda t: t.cpu().view(torch.uint8)  # noqa: E731
    for got, w in ((kd, want[0]), (vd, want[1])):
        bad = raw(got) != raw(w)
        if kind == "fp8":  # NaN has two codes
            bad &= ~((raw(got) & 0x7F == 0x7F) & (raw(w) & 0x7F == 0x7F))
        assert not bool(bad.any())
    for got, w in ((ksd, want_s[0]), (vsd, want_s[1])):
        assert w is None or torch.equal(got.cpu(), w)
    # Read back: rows of 0, 1, some and all positions of a table.
    width = pool
    table = torch.stack([torch.randperm(pool, generator=g) for _ in range(4)]).to(torch.int32)
    lens = [0, 1, min(width * page, page + 1), width * page]
    off = [0]
    for m in lens:
        off.append(off[-1] + m)
    for out in ([torch.bfloat16, torch.float32] if kind == "fp8" else [DT[dtype]]):
        kb, vb = kernels.paged_kv_read(kd, vd, dev(table), dev(torch.tensor(off)), off[-1] + 2, k_scale=ksd, v_scale=vsd,
                                       dtype=out)
        for got, pages, s in ((kb, want[0], want_s[0]), (vb, want[1], want_s[1])):
            val = pu.dequantise(pages, s) if kind == "fp8" else pages
            flat = [val[table[r].long()].transpose(1, 2).reshape(-1, kv, dim)[:m] for r, m in enumerate(lens)]
            w = torch.cat(flat + [torch.zeros(2, kv, dim, dtype=val.dtype)]).to(out)
            assert torch.equal(torch.nan_to_num(got.cpu(), 7.0), torch.nan_to_num(w, 7.0))
    assert kernels.read_status() == 0


def test_write_of_values_that_are_not_finite():
    """Infinities and NaN are held as NaN and leave the scale to the finite values."""
    x = torch.randn(2, 3, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    x[0, 2, 5], x[0, 2, 6], x[1, 2, 7] = float("inf"), float("nan"), float("-inf")
    k = torch.zeros(1, 1, 2, 64, dtype=torch.float8_e4m3fn, device=DEV)
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(1, 1, 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    cs = torch.zeros(1, 32, 2, device=DEV)
    cs[..., 0] = 1
    idx = torch.tensor([0, 0], device=DEV)
    kernels.paged_rope_kv(x.reshape(2, -1).to(DEV), cs, idx, k, v, torch.tensor([0, 1], device=DEV), 1, 1, k_scale=ks, v_scale=vs)
    codes, e = pu.quantise(x[:, 2])
    assert torch.equal(vs.cpu()[0, 0].long(), e + 127)
    got = pu.dequantise(v.cpu()[0, 0], vs.cpu()[0, 0])
    want = pu.dequantise(codes, (e + 127).to(torch.uint8))
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x[:, 2].float()))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_write_and_read_report_bad_places():
    k, v, _, _, _, _ = pu.cache(3, 1, 4, 64, "own", torch.Generator().manual_seed(0))
    kd, vd = k.to(DEV), v.to(DEV)
    qkv = torch.ones(2, 3 * 64, dtype=torch.bfloat16, device=DEV)
    cs = torch.ones(8, 32, 2, device=DEV)
    for pos, slots in (([0, 8], [-1, -1]), ([0, -1], [-1, -1]), ([0, 0], [12, -1]), ([0, 0], [2**40, -1])):
        q = kernels.paged_rope_kv(qkv, cs, torch.tensor(pos, device=DEV), kd, vd, torch.tensor(slots, device=DEV), 1, 1)
        assert kernels.read_status() == 1
        if pos[1] != 0:
            assert bool((q[1] == 0).all())
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    off = torch.tensor([0, 5], device=DEV)
    for table in ([[0, 3]], [[0, -1]]):
        kb, _ = kernels.paged_kv_read(kd, vd, torch.tensor(table, dtype=torch.int32, device=DEV), off, 5)
        assert kernels.read_status() == 1
        assert bool((kb[4] == 0).all()) and torch.equal(kb[:4].cpu(), k[0].transpose(0, 1))
    kernels.paged_kv_read(kd, vd, torch.tensor([[0]], dtype=torch.int32, device=DEV), off, 5)  # past the table
    assert kernels.read_status() == 1


# --------------------------------------------------------------------------------------------------------------- packed

def run_packed(heads, kv, dim, new, keys, dtype, seed=0, fused=False, nan_gaps=True, scale=None, big=1.0):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(new), sum(keys)
    q_off = [sum(new[:i]) for i in range(len(new) + 1)]
    k_off = [sum(keys[:i]) for i in range(len(keys) + 1)]
    dt = DT[dtype]
    q = (big * torch.randn(tq, heads, dim, generator=g)).to(dt)
    k = torch.randn(tk, kv, dim, generator=g).to(dt)
    v = torch.randn(tk, kv, dim, generator=g).to(dt)
    s = dim**-0.5 if scale is None else scale
    want = pu.packed(q, k, v, q_off, k_off, s)
    size = pu.packed(q, k, v.abs(), q_off, k_off, s)
    if fused:  # views of one qkv buffer
        qkv = torch.cat([q.reshape(tq, -1), k.reshape(tk, -1), v.reshape(tk, -1)], 1).to(DEV)
        qd = qkv[:, : heads * dim].view(tq, heads, dim)
        kd = qkv[:, heads * dim: (heads + kv) * dim].view(tk, kv, dim)
        vd = qkv[:, (heads + kv) * dim:].view(tk, kv, dim)
    else:
        qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    off = torch.tensor(q_off, device=DEV)
    args = (qd, kd, vd, off, None if keys == new else torch.tensor(k_off, device=DEV), scale)
    got = kernels.packed_attention(*args)
    check(got, want, size, dt)
    assert torch.equal(got, kernels.packed_attention(*args)), "two calls differ"


PROMPTS = [1, 0, 130, 7, 128, 129, 127, 64, 0, 300]


@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (4, 4, 128, "bf16"), (8, 2, 128, "bf16"), (6, 2, 128, "bf16"), (16, 1, 128, "bf16"), (2, 2, 512, "bf16"), (4, 1, 512, "bf16"),
    (6, 2, 512, "bf16"), (4, 2, 64, "bf16"), (2, 1, 256, "bf16"), (3, 1, 16, "bf16"), (4, 2, 64, "f32"), (3, 3, 128, "f32"),
    (2, 1, 512, "f32"), (2, 2, 16, "f32"), (2, 2, 32, "f32"), (4, 2, 256, "f32")])
@pytest.mark.parametrize("fused", [False, True])
def test_packed_prompts(heads, kv, dim, dtype, fused):
    run_packed(heads, kv, dim, PROMPTS, PROMPTS, dtype, fused=fused)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 2, 128, "bf16"), (4, 4, 128, "bf16"), (2, 1, 512, "bf16"), (4, 2, 64, "f32"),
                                                (64, 1, 128, "bf16"), (100, 1, 128, "bf16"), (48, 1, 512, "bf16"), (130, 1, 64, "bf16"),
                                                (4, 2, 64, "bf16"), (4, 1, 256, "bf16")])
def test_packed_chunks(heads, kv, dim, dtype):
    """Chunks with keys before them, sequences with fewer keys than queries (rows that see nothing) or none."""
    new = [1, 5, 100, 33, 0, 9, 130]
    keys = [200, 5, 421, 20, 17, 0, 129]
    run_packed(heads, kv, dim, new, keys, dtype, seed=2)


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (2, 2, 512), (4, 2, 64), (2, 1, 256)])
def test_packed_long(heads, kv, dim):
    run_packed(heads, kv, dim, [1111, 64], [1111 + 700, 2000], "bf16", seed=3)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (4, 4, 128), (6, 2, 128), (2, 1, 256), (2, 2, 512), (4, 1, 512)])
def test_packed_few_rows_over_many_keys(heads, kv, dim):
    """Few units: each is cut along its keys, and its parts are added up (the last parts of short sequences are empty)."""
    run_packed(heads, kv, dim, [3, 40, 1, 7, 0, 5], [1500, 700, 2, 7, 30, 4], "bf16", seed=6)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 4, 64, "f32"), (3, 1, 128, "f32"), (2, 1, 512, "f32"), (2, 2, 256, "f32"), (4, 4, 16, "bf16"),
                                                (6, 2, 32, "bf16"), (130, 1, 64, "bf16")])
@pytest.mark.parametrize("new,keys", [([16], [1516]), ([3, 40, 1, 7, 0, 5], [1500, 700, 2, 3, 30, 4]), ([1, 20], [2600, 5])])
def test_packed_parts_without_tensor_cores(heads, kv, dim, dtype, new, keys):
    """Few queries over many keys where no tensor-core kernel takes the call: parts of the keys, some of them empty."""
    run_packed(heads, kv, dim, new, keys, dtype, seed=13)


MANY = [  # more units than CTAs; some sequences see fewer keys than queries
    (32, 4, [300, 1, 0, 65, 500, 128, 250, 16, 17], [300, 200, 3, 20, 900, 0, 251, 16, 145]),
    (60, 20, [430, 1, 300, 90], [430, 130, 260, 300]), (32, 32, [1100, 513], [1100, 600])]


@pytest.mark.parametrize("heads,kv,new,keys", MANY)
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_many_units(heads, kv, new, keys, dim):
    run_packed(heads, kv, dim, new, keys, "bf16", seed=7)


@pytest.mark.parametrize("dim", [64, 128])
def test_packed_many_units_with_large_scores(dim):
    run_packed(*MANY[0][:2], dim, *MANY[0][2:], "bf16", seed=8, big=30.0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_packed_many_units_with_hidden_values(dim, bad):
    """As test_packed_hidden_values_stay_out, where a sequence has many query tiles."""
    g = torch.Generator().manual_seed(10)
    off = [0, 600, 1300]
    q = torch.randn(1300, 32, dim, generator=g).to(torch.bfloat16)
    k = torch.randn(1300, 4, dim, generator=g).to(torch.bfloat16)
    v = torch.randn(1300, 4, dim, generator=g).to(torch.bfloat16)
    want = pu.packed(q, k, v, off, off, dim**-0.5)
    size = pu.packed(q, k, v.abs(), off, off, dim**-0.5)
    for at in (410, 600 + 690):
        k[at], v[at] = bad, bad
    got = kernels.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(off, device=DEV))
    blind = [*range(0, 410), *range(600, 1290)]
    check(got[blind], want[blind], size[blind], torch.bfloat16)
    if bad != bad:
        assert bool(torch.isnan(got[410:600]).all()) and bool(torch.isnan(got[1290:]).all())
    kernels.read_status()


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_packed_cut_units_with_hidden_values(dim):
    """As test_packed_hidden_values_stay_out, where the units are cut."""
    g = torch.Generator().manual_seed(9)
    q = torch.randn(4, 2, dim, generator=g).to(torch.bfloat16)
    k = torch.randn(900, 2, dim, generator=g).to(torch.bfloat16)
    v = torch.randn(900, 2, dim, generator=g).to(torch.bfloat16)
    off, k_off = [0, 4], [0, 900]
    want = pu.packed(q, k, v, off, k_off, dim**-0.5)
    size = pu.packed(q, k, v.abs(), off, k_off, dim**-0.5)
    k[898], v[898] = float("nan"), float("nan")
    got = kernels.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(off, device=DEV), torch.tensor(k_off, device=DEV))
    check(got[:2], want[:2], size[:2], torch.bfloat16)
    assert bool(torch.isnan(got[2:]).all())


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (512, "bf16"), (64, "f32")])
def test_packed_large_scores(dim, dtype):
    """Scores of hundreds: one key takes all, and the running maximum moves tile by tile."""
    run_packed(4, 2, dim, [150, 40], [400, 40], "bf16" if dtype == "bf16" else "f32", seed=4, big=30.0 if dtype == "bf16" else 3.0)


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (512, "bf16"), (64, "f32"), (64, "bf16"), (256, "bf16"), (32, "bf16")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_packed_hidden_values_stay_out(dim, dtype, bad):
    """What is not finite in the keys and values of a position reaches the queries that see it, and no other query and no
    other sequence."""
    g = torch.Generator().manual_seed(5)
    new, keys = [100, 70, 40], [100, 90, 40]
    q_off, k_off = [0, 100, 170, 210], [0, 100, 190, 230]
    dt = DT[dtype]
    q = torch.randn(210, 4, dim, generator=g).to(dt)
    k = torch.randn(230, 2, dim, generator=g).to(dt)
    v = torch.randn(230, 2, dim, generator=g).to(dt)
    want = pu.packed(q, k, v, q_off, k_off, dim**-0.5)
    size = pu.packed(q, k, v.abs(), q_off, k_off, dim**-0.5)
    for at in (60, 100 + 55, 190):  # position 60 of sequence 0, 55 of sequence 1 (query 35), 0 of sequence 2
        k[at], v[at] = bad, bad
    got = kernels.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(q_off, device=DEV), torch.tensor(k_off, device=DEV))
    blind = [*range(0, 60), *range(100, 135)]
    check(got[blind], want[blind], size[blind], dt)
    sees = [*range(60, 100), *range(135, 210)]
    if bad != bad:
        assert bool(torch.isnan(got[sees]).all())
    kernels.read_status()


@pytest.mark.parametrize("heads,kv,dim,dtype,lens", [
    (4, 2, 128, "bf16", [1, 130, 300]), (32, 4, 128, "bf16", [700, 600]), (32, 4, 64, "bf16", [1, 700, 600]), (4, 2, 256, "bf16", [1, 300]),
    (4, 2, 512, "bf16", [1, 300]), (4, 2, 64, "f32", [1, 130]), (4, 2, 32, "bf16", [1, 130])])
def test_packed_scores_of_minus_infinity(heads, kv, dim, dtype, lens):
    """The first key of each sequence scores -inf: a query that sees it alone has no softmax (NaN), the others leave it out."""
    g = torch.Generator().manual_seed(11)
    dt, n = DT[dtype], sum(lens)
    off = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dt) for h in (heads, kv, kv))
    q[:, :, 3] = 1.0
    k[off[:-1], :, 3] = float("-inf")
    want = pu.packed(q, k, v, off, off, dim**-0.5)
    size = pu.packed(q, k, v.abs(), off, off, dim**-0.5)
    got = kernels.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(off, device=DEV)).cpu()
    first = torch.zeros(n, dtype=torch.bool)
    first[off[:-1]] = True
    assert bool(torch.isnan(want[first]).all()) and bool(torch.isnan(got[first]).all())
    check(got[~first], want[~first], size[~first], dt)


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [
    (4, 2, 128, 16, "bf16"), (4, 4, 512, 64, "bf16"), (8, 1, 64, 16, "bf16"), (4, 1, 256, 128, "bf16"), (4, 2, 64, 16, "f32"), (4, 2, 32, 16, "bf16")])
@pytest.mark.parametrize("tokens", [1, 3])
def test_paged_scores_of_minus_infinity(heads, kv, dim, page, dtype, tokens):
    """As test_packed_scores_of_minus_infinity, over pages."""
    g = torch.Generator().manual_seed(12)
    dt, lens = DT[dtype], [1, 2, 300, 131]
    table, pool = pu.table_for([n + tokens - 1 for n in lens], page, g)
    k, v, _, _, _, _ = pu.cache(pool, kv, page, dim, "own", g, dt)
    q = torch.randn(len(lens) * tokens, heads, dim, generator=g).to(dt)
    q[:, :, 3] = 1.0
    k[table[:, 0].long(), :, 0, 3] = float("-inf")
    length = torch.tensor(lens)
    want = pu.paged(q, k, v, table, length, dim**-0.5, tokens)
    size = pu.paged(q, k, v.abs(), table, length, dim**-0.5, tokens)
    got = kernels.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), length.to(DEV), dim**-0.5, tokens=tokens).cpu()
    assert bool(torch.isnan(want[0]).all()) and bool(torch.isnan(got[0]).all())
    check(got[1:], want[1:], size[1:], dt)


def test_packed_bad_offsets_are_reported():
    q = torch.randn(10, 2, 128).to(torch.bfloat16).to(DEV)
    kernels.packed_attention(q, q, q, torch.tensor([0, 4, 10], device=DEV), torch.tensor([0, 4, 11], device=DEV))
    assert kernels.read_status() == 1
    kernels.packed_attention(q, q, q, torch.tensor([-1, 4, 10], device=DEV), torch.tensor([0, 4, 10], device=DEV))
    assert kernels.read_status() == 1


def test_refusals_of_the_c_entries():
    """What only the library's own checks see."""
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    n = torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="heads"):
        kernels.paged_attention(q[:, :3].contiguous(), k, k, table, n, 1.0)
    with pytest.raises(ValueError, match="head_dim"):
        k96 = torch.zeros(4, 2, 16, 96, dtype=torch.bfloat16, device=DEV)
        kernels.paged_attention(q[:, :, :96].contiguous(), k96, k96, table, n, 1.0)
    odd = torch.zeros(4 * 2 * 16 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, 2, 16, 128)
    with pytest.raises(ValueError, match="aligned"):
        kernels.paged_attention(q, odd, odd, table, n, 1.0)
    loose = torch.zeros(4, 2, 16, 132, dtype=torch.bfloat16, device=DEV)[..., :128]
    with pytest.raises(ValueError, match="strides"):
        kernels.paged_attention(q, loose, loose, table, n, 1.0)
    with pytest.raises(ValueError, match="strides"):
        kernels.packed_attention(loose[0].transpose(0, 1), k[0].transpose(0, 1), k[0].transpose(0, 1), n)
    with pytest.raises(ValueError, match="heads"):
        kernels.packed_attention(q[:, :3], k[0, :, :2].contiguous(), k[0, :, :2].contiguous(), n)


@pytest.mark.parametrize("kind", ["own", "fp8"])
def test_on_another_stream_and_in_a_graph(kind):
    """The chain on a side stream, then captured and replayed with new lengths: grids depend on host sizes only."""
    g = torch.Generator().manual_seed(11)
    page, heads, kv, dim, rows = 16, 8, 2, 128, 3
    lens = [33, 100, 7]
    table, pool = pu.table_for([200] * rows, page, g)
    k, v, ks, vs, _, _ = pu.cache(pool, kv, page, dim, kind, g)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    kd, vd, ksd, vsd, td = dev(k), dev(v), dev(ks), dev(vs), dev(table)
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).to(DEV)
    ang = torch.rand(256, dim // 2, generator=g)
    cs = torch.stack([ang.cos(), ang.sin()], -1).to(DEV)
    pos = torch.tensor(lens, device=DEV)

    def step():
        slots = td.gather(1, pos[:, None] // page)[:, 0].long() * page + pos % page
        q = kernels.paged_rope_kv(qkv, cs, pos, kd, vd, slots, heads, kv, k_scale=ksd, v_scale=vsd)
        return kernels.paged_attention(q, kd, vd, td, pos + 1, dim**-0.5, k_scale=ksd, v_scale=vsd)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for shift in (0, 5, 60):
        pos.copy_(torch.tensor(lens, device=DEV) + shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())
    assert kernels.read_status() == 0
