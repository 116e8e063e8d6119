"""Attention over one 4-bit page of so many positions that a position's place in it passes 32 bits."""

import pytest
import torch

import int4_util as iu
from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu


def test_a_page_past_32_bits():
    """2^24 positions of zeros (bytes that other scales would make values of), then 40 that the query prefers by 40 and more: those
    alone count (the others' weights are 2^24 e^-40 < 2^-33 in all), and the first keys' bytes are not read in their place. Bound as
    in test_int4_cache_gpu.py, the sums' part for 40 keys."""
    dim, page, first, n = 512, 1 << 25, 1 << 24, 40
    g = torch.Generator().manual_seed(0)
    q = torch.randn(1, 1, dim, generator=g).bfloat16()
    x = 2.5 * q[0].float() + 0.3 * torch.randn(n, dim, generator=g)  # scores of about 2.5 * 512 * 512^-0.5 = 57
    kc, ks = iu.quantise(x.bfloat16())
    vc, vs = iu.quantise(torch.randn(n, dim, generator=g).bfloat16())
    kval, vval = iu.values(kc, ks).double(), iu.values(vc, vs).double()
    scores = kval @ q[0, 0].double() * dim**-0.5
    assert float(scores.min()) > 40
    p = torch.softmax(scores, 0)
    want = p @ vval
    size = p @ vval.abs(), (p @ vs.double().abs()).repeat_interleave(32)
    shape = (1, 1, page)
    k, v = (torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    kscale, vscale = (torch.zeros(*shape, dim // 32, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = slice(first, first + n)
    k[0, 0, at], v[0, 0, at] = iu.pack(kc, True).cuda(), iu.pack(vc, False).cuda()
    kscale[0, 0, at], vscale[0, 0, at] = ks.cuda(), vs.cuda()
    got = kernels.paged_attention(q.cuda(), k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([first + n], device="cuda"),
                                  dim**-0.5, k_scale=kscale, v_scale=vscale)[0, 0].double().cpu()
    bound = 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-10) * size[0] + 2.0**-11 * size[1]
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1, worst
    assert kernels.read_status() == 0
