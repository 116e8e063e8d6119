"""Plain forms in 64 bits of the paged-cache operators and the packed-prompt attention, and inputs for their tests."""

from __future__ import annotations

import torch


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, e) of the vectors x [..., D]: e the smallest integer with max|x| <= 448 * 2^e over the finite values, held
    to [-40, 40]; codes x * 2^-e rounded to e4m3, NaN for what is not finite or lies past 448 * 2^40."""
    x = x.double()
    amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(amax.shape, -40, dtype=torch.int64)
    for i in range(-40, 40):
        e = torch.where(amax > 448.0 * 2.0**i, torch.full_like(e, i + 1), e)
    y = x * 2.0 ** -e.double()[..., None]
    y = torch.where(y.abs() <= 448.0, y, torch.full_like(y, float("nan")))
    return y.float().to(torch.float8_e4m3fn), e


def dequantise(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return codes.float() * 2.0 ** (scale.float() - 127.0)[..., None]


def rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor, scale: float) -> torch.Tensor:
    """Attention of query i over the first seen[i] keys only (the others are not even looked at), in float64."""
    out = torch.zeros(q.size(0), v.size(1), dtype=torch.float64)
    for i in range(q.size(0)):
        n = max(0, min(int(seen[i]), k.size(0)))
        if n:
            x = (k[:n].double() @ q[i].double()) * scale
            p = torch.exp(x - x.max())
            out[i] = (p / p.sum()) @ v[:n].double()
    return out


def packed(q, k, v, q_off, k_off, scale):
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    heads, kv = q.size(1), k.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64)
    for s in range(len(q_off) - 1):
        a, b, c, d = q_off[s], q_off[s + 1], k_off[s], k_off[s + 1]
        seen = torch.arange(1, b - a + 1) + (d - c) - (b - a)
        for h in range(heads):
            j = h // (heads // kv)
            out[a:b, h] = rows(q[a:b, h], k[c:d, j], v[c:d, j], seen, scale)
    return out


def paged(q, k_pages, v_pages, table, lengths, scale, tokens):
    """k_pages / v_pages as the numbers they stand for."""
    q, k_pages, v_pages, table = q.cpu(), k_pages.cpu(), v_pages.cpu(), table.cpu().long()
    heads, kv = q.size(1), k_pages.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64)
    for r, n in enumerate(lengths.tolist()):
        seen = n + torch.arange(tokens)
        for h in range(heads):
            j = h // (heads // kv)
            kk, vv = k_pages[table[r], j].flatten(0, 1), v_pages[table[r], j].flatten(0, 1)
            out[r * tokens:(r + 1) * tokens, h] = rows(q[r * tokens:(r + 1) * tokens, h], kk, vv, seen, scale)
    return out


def table_for(lens, page, gen, spare=2):
    """(table [rows, width] int32, pages in the pool): every row's pages anywhere in the pool."""
    counts = [-(-n // page) for n in lens]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen)
    table = torch.zeros(len(lens), max(1, max(counts)), dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c].to(torch.int32)
        at += c
    return table, total


def cache(pages, kv, page, dim, kind, gen, dtype=torch.bfloat16):
    """Random pages on the CPU: (k, v, k_scale, v_scale, k values, v values)."""
    out, values, scales = [], [], []
    for _ in range(2):
        x = torch.randn(pages, kv, page, dim, generator=gen) * torch.exp(0.7 * torch.randn(pages, kv, page, 1, generator=gen))
        x = x.to(dtype)
        if kind == "fp8":
            codes, e = quantise(x)
            scale = (e + 127).to(torch.uint8)
            out.append(codes)
            scales.append(scale)
            values.append(dequantise(codes, scale))
        else:
            out.append(x)
            scales.append(None)
            values.append(x)
    return out[0], out[1], scales[0], scales[1], values[0], values[1]


def rope(x, cs):
    """Interleaved pairs of x [N, H, D] (float32 products, each rounded) turned by cs [N, D/2, 2]; x's dtype."""
    f = x.float()
    re, im = f[..., 0::2], f[..., 1::2]
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([re * co - im * si, re * si + im * co], -1).flatten(-2).to(x.dtype)
