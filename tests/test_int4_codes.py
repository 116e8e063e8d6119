"""The 4-bit append's codes of bf16 values, a product with the scale's reciprocal rounded to multiples of 2^-14 first, against those of an
fp32 division: for every pair of significands (8 bits each) and every quotient from 2^-12 to 8, of both signs."""

import numpy as np
import pytest
import torch

import int4_util as iu

EXPONENTS = range(-12, 4)  # of the value over the scale's; quotients under 2^-1 have the code of 0


def test_reciprocal_gives_the_divisions_codes():
    """Reciprocals off by up to 3 units in the last place (the device's are within 2)."""
    x, s = np.meshgrid(np.arange(128, 256, dtype=np.float32), np.arange(128, 256, dtype=np.float32))
    for d in EXPONENTS:
        for sign in (1.0, -1.0):
            v = (x * np.float32(sign * 2.0**d)).astype(np.float32)
            keep = np.abs(v / s) < 8.04  # (the largest of a group is 8 scales, but for the scale's rounding)
            want = np.clip(np.rint(v / s), -8, 7) + 8
            base = (np.float32(1) / s).astype(np.float32)
            for ulps in range(-3, 4):
                inv = (base.view(np.int32) + ulps).view(np.float32)
                q = (v * inv + np.float32(768)) - np.float32(768)
                assert q.dtype == np.float32
                c = np.clip(q, np.float32(-8), np.float32(7)) + np.float32(12582920)
                assert np.array_equal((c.view(np.int32) & 15)[keep], want[keep])


@pytest.mark.gpu
def test_every_pair_on_the_gpu():
    """Groups whose largest value has each significand, the others every value beside it."""
    from omniasr_b200 import kernels

    x = torch.arange(128, 256, dtype=torch.float32)
    others = torch.cat([x * 2.0**d for d in EXPONENTS])  # relative to a scale with a significand of 128 to 255
    others = torch.cat([others, -others])
    groups = []
    for s in range(128, 256):
        top = 8.0 * s
        v = others[others.abs() <= top]
        v = torch.cat([v, torch.zeros(-v.numel() % 31)]).view(-1, 31)
        groups.append(torch.cat([torch.full((v.size(0), 1), -top), v], 1))
    v = torch.cat(groups)
    v = torch.cat([v, torch.zeros(-v.size(0) % 16, 32)]).reshape(-1, 1, 512).bfloat16()  # [tokens, one head, 16 groups]
    assert torch.equal(v.float().flatten(), torch.cat([torch.cat(groups).flatten(), torch.zeros(v.numel() - 32 * sum(map(len, groups)))]))
    n = v.size(0)
    for scale in (1.0, -1.0, 2.0**-60, 2.0**60, -(2.0**-107), -(2.0**-108)):  # (the last two: just above and below the product's least scale, 2^-100)
        data = (v * scale).bfloat16()
        qkv = torch.cat([torch.zeros(n, 2, 512, dtype=torch.bfloat16), data], 1).reshape(n, -1).cuda()
        k, kept = (torch.zeros(n, 1, 1, 256, dtype=torch.uint8, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros(n, 1, 1, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        cs = torch.ones(1, 256, 2, device="cuda")
        kernels.paged_rope_kv(qkv, cs, torch.zeros(n, dtype=torch.int64, device="cuda"), k, kept, torch.arange(n, device="cuda"), 1, 1,
                              k_scale=ks, v_scale=vs)
        codes, s = iu.quantise(data)
        assert torch.equal(vs.cpu()[:, 0], s)
        assert torch.equal(iu.unpack(kept.cpu()[:, 0], False), codes)
    assert kernels.read_status() == 0
