"""The 4-bit form of a paged cache's vectors in plain operations, and inputs for its tests."""

from __future__ import annotations

import torch

import paged_util as pu


def order(dim: int, keys: bool) -> torch.Tensor:
    """Where dim d's code lies among a vector's (low four bits of a byte first)."""
    at = []
    for d in range(dim):
        u = d // 4
        groups, g, i = min(4, dim // 32), u % 32 // 8, u % 8
        word = (i // 2 * groups + g) * 2 + i % 2 if keys else i * groups + g
        at.append(4 * (u // 32 * 32 + word) + d % 4)
    return torch.tensor(at)


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes 0..15 [..., D] by dim, scales bf16 [..., D / 32]) of the vectors x."""
    g = x.float().unflatten(-1, (-1, 32))
    finite = torch.isfinite(g).all(-1)
    safe = torch.where(finite[..., None], g, torch.zeros_like(g))
    lo, hi = safe.amin(-1), safe.amax(-1)
    s = (torch.where(hi > -lo, hi, lo) * -0.125).bfloat16()
    f = s.float()[..., None]
    c = torch.where(f == 0, torch.zeros_like(safe), safe / f).round().clamp(-8, 7) + 8
    return c.to(torch.uint8).flatten(-2), torch.where(finite, s, torch.full_like(s, float("nan")))


def values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What codes (by dim) and scales stand for (fp32, exact)."""
    return ((codes.float() - 8).unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


def pack(codes: torch.Tensor, keys: bool) -> torch.Tensor:
    stored = torch.empty_like(codes)
    stored[..., order(codes.size(-1), keys).to(codes.device)] = codes
    return stored[..., 0::2] | stored[..., 1::2] << 4


def unpack(data: torch.Tensor, keys: bool) -> torch.Tensor:
    c = torch.stack([data & 15, data >> 4], -1).flatten(-2)
    return c[..., order(c.size(-1), keys).to(c.device)]


def cache(pages, kv, page, dim, gen):
    """Random pages on the CPU: (k, v, k_scale, v_scale, k values, v values)."""
    out = []
    for keys in (True, False):
        x = torch.randn(pages, kv, page, dim, generator=gen) * torch.exp(0.7 * torch.randn(pages, kv, page, 1, generator=gen))
        codes, scale = quantise(x.bfloat16())
        out.append((pack(codes, keys), scale, values(codes, scale)))
    (k, ks, kval), (v, vs, vval) = out
    return k, v, ks, vs, kval, vval


def paged_want(q, kval, vval, vs, table, length, scale, tokens):
    """(o, (sum p |v| / sum p, sum p |s| / sum p with each group's scale s)) in float64."""
    groups = vs.float().abs().repeat_interleave(32, -1)
    return (pu.paged(q, kval, vval, table, length, scale, tokens),
            (pu.paged(q, kval, vval.abs(), table, length, scale, tokens), pu.paged(q, kval, groups, table, length, scale, tokens)))
