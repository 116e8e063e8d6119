"""The serving example end to end: prompts prefilled from pages in chunks and decoded together, against attention in float32
without a cache. A token may differ only where that form holds the two nearly equal: its own bf16 roundings move a logit by
some 2^-6 (products of 512 and 256 terms through two layers), an 8-bit cache's rounding of keys and values by some 2^-3."""

import sys

import pytest
import torch

from conftest import ROOT
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,gap", [(torch.bfloat16, 0.1), (torch.float8_e4m3fn, 0.6)])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 8), (2, 2, 512, 64)])
def test_serving_example(kind, gap, heads, kv, dim, page):
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import paged_serving as ps
    finally:
        sys.path.pop(0)
    model = ps.Decoder(heads=heads, kv_heads=kv, dim=dim)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 200, 1, 63, 64)]
    out = ps.serve(model, prompts, 8, kind, page=page)
    for prompt, tokens in zip(prompts, out):
        assert len(tokens) == 9
        for _, behind in ps.dense(model, prompt, tokens):
            assert behind <= gap
    assert kernels.read_status() == 0


def test_drafts_over_pages_equal_single_tokens():
    """Four draft tokens in one step see what they see one at a time (bf16 pages: the same keys, the same attention up to its
    rounding)."""
    from omniasr_b200.paged import PagedCache

    g = torch.Generator().manual_seed(3)
    heads, kv, dim, n = 8, 2, 128, 4
    cs = torch.ones(512, dim // 2, 2, device="cuda")
    cs[..., 1] = 0
    qkv = torch.randn(2 * 100 + 2 * n, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).cuda()
    got = []
    for drafts in (True, False):
        c = PagedCache(1, 40, 16, kv, dim)
        seqs = [c.add(), c.add()]
        c.prefill(0, qkv[:200], cs, c.extend(seqs, [100, 100]), heads)
        new = qkv[200:].view(2, n, -1)
        if drafts:
            got.append(c.decode(0, new.reshape(2 * n, -1), cs, c.extend(seqs, [n, n]), heads).view(2, n, heads, dim))
        else:
            got.append(torch.stack([c.decode(0, new[:, i].contiguous(), cs, c.extend(seqs, [1, 1]), heads) for i in range(n)], 1))
    assert float((got[0].float() - got[1].float()).abs().max()) <= 2e-2
    assert kernels.read_status() == 0
