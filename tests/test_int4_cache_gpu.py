"""The 4-bit paged cache on the GPU: write, read back and attention, and the norms of queries and keys with the append.

Writes and read-backs of paged_rope_kv are exact (the rotation is rounded as the plain form rounds it, the codes are one fp32
division). Attention, bf16: the output's rounding is at most 2^-8 |o|; a probability times its group's scale s is rounded once, to
fp16, by 2^-11 of it: 2^-11 A with A = sum p |v| / sum p; the scores' products and sums, the exponential and the weights' sum stay well
under 2^-10 A. The sums of products with the codes c and with their offset, each at most 15 B with B = sum p |s| / sum p, are kept in
fp32: two steps per 16 keys and warp, at least 4 warps, each off by at most 2^-23 of 15 B, for at most 5000 keys 158 x 15 x 2^-23 B <
2^-11 B. fp32: 2e-5 (1 + |o|), the framework's own.
Norms: the sum of squares takes at most 21 roundings (16 terms a lane, 5 steps of a shuffle), which the root halves, the root
itself 4 half steps, the two products, the rotation's and its sum 4: under 32 x 2^-24 = 2^-19 of the terms that a rotation adds,
and the one rounding to the type."""

import pytest
import torch

import int4_util as iu
import paged_util as pu
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731


def check(got, want, size, dtype):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), "not finite"
    if dtype == torch.float32:
        bound = 2e-5 * (1 + want.abs())
    else:
        bound = 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-10) * size[0] + 2.0**-11 * size[1] + 1e-30
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} past the bound; worst " \
                                f"{float(((got - want).abs() / bound).max()):.3g} times"
    assert kernels.read_status() == 0


def spoil(k, v, ks, vs, table, lens, page):
    """NaN scales and other codes at every position that no row's length covers."""
    used = torch.zeros(k.size(0), page, dtype=torch.bool)
    for r, n in enumerate(lens):
        for j in range(n):
            used[int(table[r, j // page]), j % page] = True
    for t, x in ((k, 0xA5), (v, 0x5A), (ks, float("nan")), (vs, float("nan"))):
        t.permute(0, 2, 1, 3)[~used] = x


def inputs(heads, kv, dim, page, lens, tokens, dtype, seed=0, spare=2):
    g = torch.Generator().manual_seed(seed)
    covered = [max(0, n + tokens - 1) for n in lens]
    table, pool = pu.table_for(covered, page, g, spare)
    k, v, ks, vs, kval, vval = iu.cache(pool, kv, page, dim, g)
    q = torch.randn(len(lens) * tokens, heads, dim, generator=g).to(DT[dtype])
    return g, covered, table, k, v, ks, vs, kval, vval, q


def run_paged(heads, kv, dim, page, lens, tokens, dtype, seed=0, layout="page", scale=None):
    _, covered, table, k, v, ks, vs, kval, vval, q = inputs(heads, kv, dim, page, lens, tokens, dtype, seed)
    scale = dim**-0.5 if scale is None else scale
    length = torch.tensor(lens)
    want, size = iu.paged_want(q, kval, vval, vs, table, length, scale, tokens)
    spoil(k, v, ks, vs, table, covered, page)
    k, v = dev(k), dev(v)
    if layout == "token":  # [pages, page, kv, D / 2] storage
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif layout == "both":  # K and V of a page side by side
        both = torch.stack([k, v], 1)
        k, v = both[:, 0], both[:, 1]
    call = lambda: kernels.paged_attention(dev(q), k, v, dev(table), dev(length), scale, tokens=tokens, k_scale=dev(ks),  # noqa: E731
                                           v_scale=dev(vs))
    got = call()
    check(got, want, size, DT[dtype])
    assert torch.equal(got, call()), "two calls differ"


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300, 511, 700]
SHAPES = [(8, 2, 128, 16, "bf16"), (4, 4, 128, 64, "bf16"), (6, 2, 128, 8, "bf16"), (32, 1, 128, 32, "bf16"), (16, 1, 128, 128, "bf16"),
          (4, 4, 512, 64, "bf16"), (8, 1, 512, 16, "bf16"), (4, 2, 256, 16, "bf16"), (3, 3, 64, 16, "bf16"), (4, 1, 128, 12, "bf16"),
          (4, 2, 128, 256, "bf16"), (2, 2, 32, 4, "bf16"), (8, 2, 64, 32, "bf16"), (16, 1, 64, 128, "bf16"), (20, 1, 256, 64, "bf16"),
          (2, 1, 128, 1, "bf16"), (4, 2, 64, 16, "f32"), (3, 1, 128, 16, "f32"), (2, 2, 512, 8, "f32"), (4, 4, 32, 5, "f32"),
          (8, 1, 256, 16, "f32")]


@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("heads,kv,dim,page,dtype", SHAPES)
def test_attention_lengths(heads, kv, dim, page, dtype, tokens):
    run_paged(heads, kv, dim, page, LENS, tokens, dtype, seed=heads * dim + page)


@pytest.mark.parametrize("layout", ["token", "both"])
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_attention_strides(layout, dim):
    run_paged(4, 2, dim, 16, [1, 40, 0, 97], 1, "bf16", seed=dim, layout=layout)


@pytest.mark.parametrize("heads,kv,dim,tokens", [(32, 8, 128, 5), (32, 8, 128, 8), (8, 1, 128, 1), (24, 8, 64, 7), (8, 8, 512, 5), (16, 1, 256, 2),
                                                 (9, 1, 128, 1), (40, 1, 128, 2)])
def test_attention_drafts(heads, kv, dim, tokens):
    run_paged(heads, kv, dim, 16, [3, 0, 250, 64, 65], tokens, "bf16", seed=tokens + dim)


@pytest.mark.parametrize("rows,n,heads,kv,dim,page", [(1, 5000, 8, 1, 128, 16), (2, 3001, 16, 4, 128, 64), (1, 2500, 2, 2, 512, 32), (1, 4097, 4, 4, 64, 8),
                                                       (150, 40, 4, 2, 128, 16), (300, 9, 2, 2, 64, 8), (3, 2048, 8, 8, 256, 128)])
def test_attention_few_long_and_many_short_rows(rows, n, heads, kv, dim, page):
    run_paged(heads, kv, dim, page, [max(0, n - 7 * i) for i in range(rows)], 1, "bf16", seed=n)


@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_attention_scales(scale):
    run_paged(8, 2, 128, 16, [1, 200, 33], 2, "bf16", seed=5, scale=scale)


def test_attention_of_queries_of_all_sizes():
    """Queries of very different sizes share a kv head; tiny and large ones keep their softmax."""
    _, covered, table, k, v, ks, vs, kval, vval, q = inputs(8, 1, 128, 16, [200, 31], 1, "bf16", 3)
    for h, e in enumerate([-100, -40, -20, -8, 0, 2, 4, 6]):
        q[:, h] *= 2.0**e
    length = torch.tensor([200, 31])
    want, size = iu.paged_want(q, kval, vval, vs, table, length, 0.2, 1)
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(length), 0.2, k_scale=dev(ks), v_scale=dev(vs))
    check(got, want, size, torch.bfloat16)


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (512, "bf16"), (64, "f32")])
def test_values_that_are_not_finite(dim, dtype):
    """A group that is NaN makes NaN of what sees it and of nothing else: a key the row, a value its group's 32 dims; a later
    draft's is not seen by the queries before it."""
    heads, kv, page, tokens, lens = 4, 2, 16, 3, [70, 20, 48, 5]
    _, covered, table, k, v, ks, vs, kval, vval, q = inputs(heads, kv, dim, page, lens, tokens, dtype, 9)
    length = torch.tensor(lens)
    want, size = iu.paged_want(q, kval, vval, vs, table, length, 0.1, tokens)
    spoil(k, v, ks, vs, table, covered, page)
    at = lambda r, j: (int(table[r, j // page]), j % page)  # noqa: E731
    hide = torch.zeros(len(lens) * tokens, heads, dim, dtype=torch.bool)
    p, o = at(0, 33)
    ks[p, 0, o, 1] = float("nan")  # row 0: a key of kv head 0
    hide[0:3, 0:2] = True
    p, o = at(1, 7)
    vs[p, 1, o, 0] = float("nan")  # row 1: a value of kv head 1, dims 0 .. 31
    hide[3:6, 2:4, :32] = True
    p, o = at(2, 48 + 1)  # row 2: the last draft's own value, seen by the last query alone
    vs[p, 0, o, dim // 32 - 1] = float("nan")
    hide[8, 0:2, dim - 32:] = True
    p, o = at(3, 5 + 1)  # row 3: the last draft's key
    ks[p, 1, o, 0] = float("nan")
    hide[11, 2:4] = True
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(length), 0.1, tokens=tokens, k_scale=dev(ks),
                                  v_scale=dev(vs)).cpu()
    assert bool(torch.isnan(got[hide]).all())
    check(torch.where(hide, torch.zeros_like(got), got), torch.where(hide, torch.zeros_like(want), want), size, DT[dtype])
    # a query that is NaN
    q[1, 1, 3] = float("nan")
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(length), 0.1, tokens=tokens, k_scale=dev(ks),
                                  v_scale=dev(vs)).cpu()
    hide[1, 1] = True
    assert bool(torch.isnan(got[hide]).all()) and bool(torch.isfinite(got[~hide]).all())


def test_bad_pages_are_reported_and_skipped():
    _, covered, table, k, v, ks, vs, kval, vval, q = inputs(8, 2, 128, 16, [60, 60], 1, "bf16", 11)
    table[1, 2] = k.size(0)
    length = torch.tensor([60, 60])
    want, size = iu.paged_want(q[:1], kval, vval, vs, table[:1], length[:1], 0.1, 1)
    got = kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(length), 0.1, k_scale=dev(ks), v_scale=dev(vs))
    assert kernels.read_status() == 1
    check(got[:1], want, size, torch.bfloat16)
    long = torch.tensor([60, 2**40])
    table[1, 2] = 0
    kernels.paged_attention(dev(q), dev(k), dev(v), dev(table), dev(long), 0.1, k_scale=dev(ks), v_scale=dev(vs))
    assert kernels.read_status() == 1


# ---------------------------------------------------------------------------------------------------------------- write, read

def append_inputs(n, heads, kv, dim, page, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    pages = -(-n // page) + 3
    x = torch.randn(n, heads + 2 * kv, dim, generator=g) * torch.exp(torch.randn(n, heads + 2 * kv, 1, generator=g))
    pos = torch.randint(0, 500, (n,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:n]
    angle = torch.arange(500)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    cs = torch.stack([angle.cos(), angle.sin()], -1).float()
    return g, pages, x.to(DT[dtype]), pos, slots, cs


@pytest.mark.parametrize("n,heads,kv,dim,page,dtype", [
    (1, 4, 4, 128, 16, "bf16"), (5, 6, 2, 64, 8, "bf16"), (40, 8, 8, 512, 64, "bf16"), (33, 4, 1, 32, 5, "bf16"), (700, 32, 8, 128, 16, "bf16"),
    (9, 2, 1, 256, 32, "bf16"), (37, 4, 2, 64, 16, "f32"), (3, 2, 2, 512, 16, "f32"), (21, 3, 1, 32, 8, "f32"), (300, 8, 2, 128, 16, "f32")])
def test_write_and_read_back(n, heads, kv, dim, page, dtype):
    g, pages, x, pos, slots, cs = append_inputs(n, heads, kv, dim, page, dtype, n + dim)
    if n > 4:
        x[2, heads, 3] = float("inf")
        x[3, heads + kv, dim - 1] = float("nan")
        x[1, heads + kv] = 0
        x[4, heads + kv, :32] = torch.tensor([2.0**-133, -(2.0**-133)] * 16).to(x.dtype)
        slots[0] = -1
    k, v = (torch.full((pages, kv, page, dim // 2), 0x3C, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.full((pages, kv, page, dim // 32), 7.0, dtype=torch.bfloat16) for _ in range(2))
    turned = pu.rope(x[:, : heads + kv], cs[pos])
    want = []
    for keys, rows, data, scale in ((True, turned[:, heads:], k, ks), (False, x[:, heads + kv:], v, vs)):
        codes, s = iu.quantise(rows)
        on = slots >= 0
        at, off = slots[on] // page, slots[on] % page
        data, scale = data.clone(), scale.clone()
        data[at, :, off] = iu.pack(codes, keys)[on]
        scale[at, :, off] = s[on]
        want.append((data, scale))
    kd, vd, ksd, vsd = dev(k), dev(v), dev(ks), dev(vs)
    q = kernels.paged_rope_kv(dev(x.reshape(n, -1)), dev(cs), dev(pos), kd, vd, dev(slots), heads, kv, k_scale=ksd, v_scale=vsd)
    assert torch.equal(q.cpu(), turned[:, :heads])
    for (data, scale), gd, gs in zip(want, (kd, vd), (ksd, vsd)):
        gs, gd = gs.cpu(), gd.cpu()
        assert torch.equal(torch.isnan(gs), torch.isnan(scale)) and torch.equal(torch.nan_to_num(gs), torch.nan_to_num(scale))
        live = ~torch.isnan(scale).repeat_interleave(32, -1)  # (a NaN group's codes stand for nothing)
        for keys in (True, False):
            if data is want[0 if keys else 1][0]:
                assert torch.equal(iu.unpack(gd, keys)[live], iu.unpack(data, keys)[live])
    # the whole pool as three rows of the table, in the model's types
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].repeat(2, 1)
    off = [0, pages * page - 3, pages * page - 3 + 2]
    for out in (torch.bfloat16, torch.float32):
        kk, vv = kernels.paged_kv_read(kd, vd, dev(table), torch.tensor(off, device=DEV), off[-1] + 2, k_scale=ksd, v_scale=vsd, dtype=out)
        for (data, scale), got, keys in zip(want, (kk, vv), (True, False)):
            rows = iu.values(iu.unpack(data, keys), scale)[table[0].long()].permute(0, 2, 1, 3).reshape(-1, kv, dim).to(out)
            rows = torch.cat([rows[: off[1]], rows[:2], torch.zeros(2, kv, dim, dtype=out)])
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=9e9), torch.nan_to_num(rows, nan=9e9))
    assert kernels.read_status() == 0


# ---------------------------------------------------------------------------------------------------------------- norms

@pytest.mark.parametrize("kind", ["own", "fp8", "int4"])
@pytest.mark.parametrize("n,heads,kv,dim,page,dtype", [
    (1, 4, 4, 128, 16, "bf16"), (5, 6, 2, 64, 8, "bf16"), (40, 8, 8, 512, 64, "bf16"), (33, 4, 1, 32, 5, "bf16"), (700, 32, 8, 128, 16, "bf16"),
    (9, 2, 1, 256, 32, "bf16"), (6, 3, 1, 16, 8, "bf16"), (37, 4, 2, 64, 16, "f32"), (3, 2, 2, 512, 16, "f32"), (21, 3, 1, 16, 8, "f32")])
def test_norm_rope_append(n, heads, kv, dim, page, dtype, kind):
    if kind == "int4" and dim < 32:
        pytest.skip("groups of 32 dims")
    g, pages, x, pos, slots, cs = append_inputs(n, heads, kv, dim, page, dtype, n + dim)
    x[0, 0] = 0
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=g)).to(x.dtype) for _ in range(2))
    eps = 1e-5
    f = x[:, : heads + kv].double()
    w = torch.cat([qw.double().expand(heads, dim), kw.double().expand(kv, dim)])
    f = f / (f.square().mean(-1, keepdim=True) + eps).sqrt() * w
    re, im = f[..., 0::2], f[..., 1::2]
    co, si = (cs[pos][:, None, :, i].double() for i in range(2))
    want = torch.stack([re * co - im * si, re * si + im * co], -1).flatten(-2)
    size = torch.stack([(re * co).abs() + (im * si).abs(), (re * si).abs() + (im * co).abs()], -1).flatten(-2)
    half = 2.0**-8 if dtype == "bf16" else 2.0**-24
    bound = half * want.abs() + 2.0**-19 * size + 1e-30
    kind_of = {"own": x.dtype, "fp8": torch.float8_e4m3fn, "int4": torch.uint8}[kind]
    shape = (pages, kv, page, dim // 2 if kind == "int4" else dim)
    k, v = (torch.zeros(shape, dtype=kind_of, device=DEV) for _ in range(2))
    ks = vs = None
    if kind == "fp8":
        ks, vs = (torch.full(shape[:-1], 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    if kind == "int4":
        ks, vs = (torch.zeros(*shape[:-1], dim // 32, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = kernels.paged_norm_rope_kv(dev(x.reshape(n, -1)), dev(qw), dev(kw), dev(cs), dev(pos), k, v, dev(slots), heads, kv, eps=eps,
                                   k_scale=ks, v_scale=vs)
    assert bool(((q.cpu().double() - want[:, :heads]).abs() <= bound[:, :heads]).all())
    at, off = dev(slots // page), dev(slots % page)
    # what the pages hold is what paged_rope_kv makes of the vectors before them: v the same bits, k within a step of its code
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    ks2, vs2 = (None, None) if ks is None else (torch.zeros_like(ks), torch.zeros_like(vs))
    kernels.paged_rope_kv(dev(x.reshape(n, -1)), dev(cs), dev(pos), k2, v2, dev(slots), heads, kv, k_scale=ks2, v_scale=vs2)
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    assert torch.equal(raw(v)[at, :, off], raw(v2)[at, :, off])
    if kind != "own":
        assert torch.equal(raw(vs)[at, :, off], raw(vs2)[at, :, off])
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    kk, _ = kernels.paged_kv_read(k, v, table, torch.tensor([0, pages * page], device=DEV), pages * page, k_scale=ks, v_scale=vs,
                                  dtype=x.dtype)
    got = kk.cpu()[slots].double()
    wk = want[:, heads:]
    if kind == "own":
        slack = bound[:, heads:]
    elif kind == "fp8":  # half a step of e4m3, 2^-4 of the value, below 2^-6 448ths of the largest 2^-10
        slack = 2.0**-4 * wk.abs() * 1.02 + bound[:, heads:] + wk.abs().amax(-1, keepdim=True) * 2.0**-16
    else:  # a step of the group's scale at most
        top = wk.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
        slack = (top / 8).expand(*top.shape[:-1], 32).flatten(-2) * 1.05 + bound[:, heads:]
    assert bool(((got - wk).abs() <= slack).all())
    assert kernels.read_status() == 0


def test_refusals():
    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype, device=DEV)  # noqa: E731
    k, s = z(4, 2, 8, 32, dtype=torch.uint8), z(4, 2, 8, 2)
    table, lengths = z(2, 2, dtype=torch.int32), z(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="head_dim"):
        kernels.paged_attention(z(2, 4, 32), k, k.clone(), table, lengths, 1.0, k_scale=s, v_scale=s)
    with pytest.raises(ValueError, match="groups are 32"):
        kernels.paged_attention(z(2, 4, 16), z(4, 2, 8, 8, dtype=torch.uint8), z(4, 2, 8, 8, dtype=torch.uint8), table, lengths, 1.0,
                                k_scale=z(4, 2, 8, 0), v_scale=z(4, 2, 8, 0))
    with pytest.raises(ValueError, match="one device"):
        kernels.paged_attention(z(2, 4, 64), k, k.clone(), table, lengths, 1.0, k_scale=s.cpu(), v_scale=s)
    odd = z(4 * 2 * 8 * 40, dtype=torch.uint8).as_strided((4, 2, 8, 32), (640, 320, 40, 1))
    with pytest.raises(ValueError, match="16-byte"):
        kernels.paged_attention(z(2, 4, 64), odd, odd, table, lengths, 1.0, k_scale=s, v_scale=s)
    flat = z(4 * 2 * 8 * 2 + 1)[1:].view(4, 2, 8, 2)
    with pytest.raises(ValueError, match="16-byte"):
        kernels.paged_attention(z(2, 4, 64), k, k.clone(), table, lengths, 1.0, k_scale=flat, v_scale=flat)
    qkv, cs, pos, w = z(3, 8 * 64), z(9, 32, 2, dtype=torch.float32), z(3, dtype=torch.int64), z(65)[1:]
    with pytest.raises(ValueError, match="16-byte"):
        kernels.paged_norm_rope_kv(qkv, w, w, cs, pos, k, k.clone(), pos, 4, 2, k_scale=s, v_scale=s.clone())
    for eps in (-1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            kernels.paged_norm_rope_kv(qkv, z(64), z(64), cs, pos, k, k.clone(), pos, 4, 2, eps=eps, k_scale=s, v_scale=s.clone())
    assert kernels.read_status() == 0


def test_norm_weights_of_the_kernel_before():
    heads, kv, dim, n = 4, 2, 128, 40
    g, pages, x, pos, slots, cs = append_inputs(n, heads, kv, dim, 16, "bf16", 5)
    w = kernels.int4_quantise(torch.randn(dim, 64, generator=g).to(DEV), 32)
    qkv, pos, slots, cs = dev(x.reshape(n, -1)), dev(pos), dev(slots), dev(cs)
    rows = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(pages, kv, 16, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def step():
        norms = kernels.decode_gemm_int4(rows, w)
        return kernels.paged_norm_rope_kv(qkv, norms[0], norms[1], cs, pos, k, v, slots, heads, kv)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step()
    for i in range(20):
        rows.copy_(torch.randn(2, 64, generator=g))
        graph.replay()
        norms = kernels.decode_gemm_int4(rows, w)
        torch.cuda.synchronize()
        got, gk = q.clone(), k.clone()
        want = kernels.paged_norm_rope_kv(qkv, norms[0], norms[1], cs, pos, k, v, slots, heads, kv)
        assert torch.equal(got, want) and torch.equal(gk, k), i
