"""4-bit weights: their layout and quantisation without a GPU, and the decode GEMM over them on one, against float64.

The GEMM's codes (c - 8) and bf16 tokens are exact operands, so the result is off by fp32 sums and the last rounding alone. With S =
sum |x W|: a chain is at most 8 steps of a block of 128 columns (each adding 16 products to the sum, whose order and truncation
count as up to 16 roundings of 2^-23), then k / 128 scaled blocks and 8 warps: (8 * 16 + k / 128 + 8) 2^-23 S < 2^-15 S for k up to 11008;
the bound used is 2^-14 S. The output's rounding is 2^-8 of the value. silu's exponential and division: 2^-20 of it, its slope is at
most 1.1."""

import dataclasses

import pytest
import torch

from omniasr_b200 import kernels

DEV = "cuda"


@pytest.mark.parametrize("n,k,group", [(13, 160, 64), (8, 128, 128), (20, 96, 32), (5, 416, 128), (1, 32, 128)])
def test_layout(n, k, group):
    g = torch.Generator().manual_seed(n * k)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = torch.rand(n, -(-k // group), generator=g).bfloat16()
    w = kernels.int4_weights(codes, scales, group)
    assert torch.equal(w.values(), (codes.float() - 8) * scales.float().repeat_interleave(group, 1)[:, :k])
    assert w.codes.shape == (-(-n // 8), -(-k // 128), 512) and w.scales.shape == (-(-n // 8), -(-k // group), 8)
    for r in range(n):  # the place that the C header documents
        for col in range(0, k, 7):
            b, c = divmod(col, 128)
            word, c = divmod(c, 32)
            lane, c = divmod(c, 8)
            at = (r % 8) * 64 + lane * 16 + word * 4
            v = int.from_bytes(bytes(w.codes[r // 8, b, at:at + 4].tolist()), "little")
            assert v >> (4 * (c // 2) + 16 * (c % 2)) & 15 == int(codes[r, col])


def test_quantise():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(24, 320, generator=g)
    x[3] = 0
    w = kernels.int4_quantise(x, 64)
    top = x.unflatten(1, (5, 64)).abs().amax(-1, keepdim=True)
    err = (w.values() - x).unflatten(1, (5, 64)).abs()
    assert bool((err <= top / 8 * 1.01).all()) and float(err.mean()) < float(top.mean()) / 28
    assert bool((w.values()[3] == 0).all())


def test_refusals():
    codes, scales = torch.zeros(8, 128, dtype=torch.uint8), torch.ones(8, 1, dtype=torch.bfloat16)
    for bad in ((codes.float(), scales, 128), (codes[:, :40], scales, 128), (codes, scales, 48), (codes, scales.float(), 128),
                (codes, scales, 64), (codes[0], scales, 128)):
        with pytest.raises(ValueError, match="int4_weights"):
            kernels.int4_weights(*bad)
    for bad in (torch.zeros(8, 40), torch.zeros(8), torch.zeros(8, 128, dtype=torch.int32)):
        with pytest.raises(ValueError, match="int4_quantise"):
            kernels.int4_quantise(bad)
    w = kernels.int4_weights(codes, scales)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="mode"):
        kernels.decode_gemm_int4(x, w, "add")
    with pytest.raises(ValueError, match="residual"):
        kernels.decode_gemm_int4(x, w, "residual")
    with pytest.raises(ValueError, match="residual"):
        kernels.decode_gemm_int4(x, w, "residual", residual=torch.zeros(3, 9, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="residual"):
        kernels.decode_gemm_int4(x, w, residual=torch.zeros(3, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="x must"):
        kernels.decode_gemm_int4(x.float(), w)
    with pytest.raises(ValueError, match="x must"):
        kernels.decode_gemm_int4(x[:, :64], w)
    with pytest.raises(ValueError, match="64 rows"):
        kernels.decode_gemm_int4(torch.zeros(65, 128, dtype=torch.bfloat16), w)
    with pytest.raises(ValueError, match="out must"):
        kernels.decode_gemm_int4(x, w, out=torch.zeros(3, 8))
    with pytest.raises(ValueError, match="gate"):
        kernels.decode_gemm_int4(x, kernels.int4_weights(codes[:7], scales[:7]), "swiglu")
    with pytest.raises(ValueError, match="CUDA"):
        kernels.decode_gemm_int4(x, w)


def case(rows, n, k, group, mode, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows + n + k)
    wr = 2 * n if mode == "swiglu" else n
    codes = torch.randint(0, 16, (wr, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = ((torch.rand(wr, -(-k // group), generator=g, device=DEV) - 0.5) * 0.02).bfloat16()
    x = torch.randn(rows, k, generator=g, device=DEV).bfloat16()
    res = torch.randn(rows, n, generator=g, device=DEV).bfloat16() if mode == "residual" else None
    return kernels.int4_weights(codes, scales, group), (codes.double() - 8) * scales.double().repeat_interleave(group, 1)[:, :k], x, res


def check(y, w, x, res, mode):
    x = x.double()
    acc, size = x @ w.t(), x.abs() @ w.abs().t()
    slack = 2.0**-14 * size
    if mode == "swiglu":
        (a, b), (ga, gb), (sa, sb) = (t.chunk(2, -1) for t in (acc, size, slack))
        s = a * torch.sigmoid(a)
        want = b * s
        slack = 1.1 * sa * b.abs() + sb * s.abs() + 1.1 * sa * sb + 2.0**-20 * want.abs()
    else:
        want = acc if res is None else acc + res.double()
        slack = slack + (0 if res is None else 2.0**-24 * res.double().abs())
    bound = 2.0**-8 * want.abs() + (1 + 2.0**-8) * slack + 1e-30
    bad = (y.double() - want).abs() > bound
    assert not bool(bad.any()), f"{int(bad.sum())} past the bound, worst {float(((y.double() - want).abs() / bound).max()):.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("rows", [1, 7, 8, 9, 16, 17, 32, 40, 64])
@pytest.mark.parametrize("n,k,group", [(4096, 4096, 128), (1000, 320, 64), (13, 160, 32), (130, 11008, 128), (5, 32, 128), (24, 2816, 64)])
def test_gemm(rows, n, k, group, mode):
    w, want, x, res = case(rows, n, k, group, mode)
    y = kernels.decode_gemm_int4(x, w, mode, residual=res)
    check(y, want, x, res, mode)
    assert torch.equal(y, kernels.decode_gemm_int4(x, w, mode, residual=res)), "two calls differ"


@pytest.mark.gpu
def test_gemm_strides_and_neighbours():
    """Rows inside wider buffers: what lies beside them is neither read nor written."""
    w, want, x, res = case(9, 77, 160, 32, "residual")
    xs = torch.full((9, 176), float("nan"), dtype=torch.bfloat16, device=DEV)
    xs[:, :160] = x
    rs = torch.full((9, 91), float("nan"), dtype=torch.bfloat16, device=DEV)
    rs[:, 3:80] = res
    ys = torch.full((11, 83), 7.0, dtype=torch.bfloat16, device=DEV)
    y = kernels.decode_gemm_int4(xs[:, :160], w, "residual", residual=rs[:, 3:80], out=ys[1:10, 2:79])
    assert y.data_ptr() == ys[1:10, 2:79].data_ptr()
    check(y, want, x, res, "residual")
    inside = torch.zeros_like(ys, dtype=torch.bool)
    inside[1:10, 2:79] = True
    assert bool((ys[~inside] == 7.0).all())
    with pytest.raises(ValueError, match="16-byte"):
        kernels.decode_gemm_int4(xs[:, 1:161], w)
    assert kernels.decode_gemm_int4(x[:0], w).shape == (0, 77)


@pytest.mark.gpu
def test_gemm_values_that_are_not_finite():
    """A token with a NaN or an infinity, and a scale that is NaN, spoil their own row and column alone."""
    w, want, x, _ = case(12, 40, 256, 64, "store")
    x[3, 200], x[9, 17] = float("nan"), float("inf")
    scales = w.scales.clone()
    scales[2, 1, 5] = float("nan")  # weight row 21
    y = kernels.decode_gemm_int4(x, kernels.Int4Weights(w.codes, scales, w.n, w.k, w.group))
    assert bool(torch.isnan(y[3]).all()) and bool((~torch.isfinite(y[9])).all()) and bool(torch.isnan(y[:, 21]).all())
    keep = [i for i in range(12) if i not in (3, 9)]
    cols = [i for i in range(40) if i != 21]
    check(y[keep][:, cols], want[cols], x[keep], None, "store")


def test_weights_of_other_sizes_are_refused():
    w = kernels.int4_weights(torch.zeros(16, 256, dtype=torch.uint8), torch.ones(16, 4, dtype=torch.bfloat16), 64)
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for bad in (dict(n=17), dict(n=24), dict(n=8), dict(group=32), dict(codes=w.codes[:1]), dict(scales=w.scales[:1]),
                dict(codes=w.codes.int()), dict(scales=w.scales.float()), dict(codes=w.codes.transpose(0, 1))):
        with pytest.raises(ValueError, match="codes and scales"):
            kernels.decode_gemm_int4(x, dataclasses.replace(w, **bad))
    with pytest.raises(ValueError, match="groups"):
        kernels.decode_gemm_int4(x, dataclasses.replace(w, group=0))
    with pytest.raises(ValueError, match="codes and scales"):
        kernels.decode_gemm_int4(torch.zeros(2, 512, dtype=torch.bfloat16), dataclasses.replace(w, k=512))


def test_out_over_an_input_is_refused():
    w = kernels.int4_weights(torch.zeros(128, 128, dtype=torch.uint8), torch.ones(128, 1, dtype=torch.bfloat16))
    buf = torch.zeros(4, 256, dtype=torch.bfloat16)
    flat = torch.zeros(2048, dtype=torch.bfloat16)
    x, y = buf[:, :128], buf[:, 128:]
    for tokens, bad in ((x, x), (x, buf[:, 64:192]), (flat[128:640].view(4, 128), flat[:512].view(4, 128))):
        with pytest.raises(ValueError, match="share memory"):
            kernels.decode_gemm_int4(tokens, w, out=bad)
    with pytest.raises(ValueError, match="share memory"):
        kernels.decode_gemm_int4(x, w, "residual", residual=flat[128:640].view(4, 128), out=flat[:512].view(4, 128))
    for mode, res in (("store", None), ("residual", y)):  # side by side, and the residual itself: the CPU is what is refused
        with pytest.raises(ValueError, match="CUDA"):
            kernels.decode_gemm_int4(x, w, mode, residual=res, out=y)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 64])
def test_residual_in_place_and_out_beside_x(rows):
    gen = torch.Generator().manual_seed(rows)
    w = kernels.int4_quantise(torch.randn(128, 128, generator=gen).to(DEV), 32)
    buf = torch.randn(rows, 256, generator=gen).bfloat16().to(DEV)
    x, y = buf[:, :128], buf[:, 128:]
    want = kernels.decode_gemm_int4(x.clone(), w, "residual", residual=y.clone())
    before = x.clone()
    got = kernels.decode_gemm_int4(x, w, "residual", residual=y, out=y)
    assert got.data_ptr() == y.data_ptr() and torch.equal(got, want) and torch.equal(x, before)
