"""The 4-bit paged cache without a GPU: its plain form against its definition, and what the wrappers refuse."""

import pytest
import torch

import int4_util as iu
from omniasr_b200 import kernels


@pytest.mark.parametrize("dim", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("keys", [True, False])
def test_order_is_a_permutation_that_unpack_undoes(dim, keys):
    assert sorted(iu.order(dim, keys).tolist()) == list(range(dim))
    codes = torch.randint(0, 16, (5, dim), dtype=torch.uint8)
    data = iu.pack(codes, keys)
    assert data.shape == (5, dim // 2) and torch.equal(iu.unpack(data, keys), codes)


def test_a_lanes_share_is_one_run_of_bytes():
    """K: lane t of 4 holds dims 8t .. 8t + 7 of each of a block's groups in 16 bytes; V: lane g of 8 dims 4g .. in 8 bytes."""
    for keys, lanes, per in ((True, 4, 8), (False, 8, 4)):
        at = iu.order(256, keys)
        for block in range(2):
            for lane in range(lanes):
                dims = [128 * block + 32 * g + per * lane + i for g in range(4) for i in range(per)]
                places = at[dims]
                n = 128 // lanes
                assert sorted(places.tolist()) == list(range(128 * block + n * lane, 128 * block + n * (lane + 1)))


def test_quantise_matches_its_definition():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(400, 64, generator=g) * torch.exp(6 * torch.randn(400, 1, generator=g))).bfloat16()
    x[0] = 0
    x[1, :32] = 1.0
    x[2, :32] = torch.tensor([3.0, -3.0] * 16).bfloat16()
    codes, scale = iu.quantise(x)
    back = iu.values(codes, scale).double()
    grp = x.double().unflatten(-1, (-1, 32))
    top = grp.abs().amax(-1)
    # half a step (an eighth of the largest), a whole one where the other end of the range is cut off
    err = (back.unflatten(-1, (-1, 32)) - grp).abs()
    assert bool((err <= (top / 8 * (1 + 2.0**-7))[..., None]).all())
    inside = (grp / scale.double()[..., None]).abs() <= 7.5
    assert bool((err[inside] <= (top / 16 * (1 + 2.0**-7))[..., None].expand_as(err)[inside]).all())
    assert bool((back[0] == 0).all()) and bool((codes[0] == 8).all())
    assert bool((scale[2, 0].float() == 0.375))  # of two as large the negative one is held exactly
    assert back[2, 1] == -3.0 and back[2, 0] == 0.375 * 7
    x[3, 5], x[3, 40] = float("inf"), float("nan")
    codes, scale = iu.quantise(x)
    assert bool(torch.isnan(scale[3]).all()) and bool(torch.isnan(iu.values(codes, scale)[3]).all())


def _cache(pages=4, kv=2, page=8, dim=64):
    k = torch.zeros(pages, kv, page, dim // 2, dtype=torch.uint8)
    s = torch.zeros(pages, kv, page, dim // 32, dtype=torch.bfloat16)
    return k, k.clone(), s, s.clone()


def test_argument_checks():
    k, v, ks, vs = _cache()
    table = torch.zeros(2, 2, dtype=torch.int32)
    lengths = torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    attend = lambda **kw: kernels.paged_attention(**{**dict(q=q, k_pages=k, v_pages=v, page_table=table, lengths=lengths,  # noqa: E731
                                                            scale=1.0, k_scale=ks, v_scale=vs), **kw})
    with pytest.raises(ValueError, match="bfloat16 scales"):
        attend(k_scale=None)
    with pytest.raises(ValueError, match="bfloat16 scales"):
        attend(v_scale=vs.float())
    with pytest.raises(ValueError, match="bfloat16 scales"):
        attend(k_scale=ks[..., :1])
    with pytest.raises(ValueError, match="bfloat16 scales"):
        attend(k_scale=ks.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="same strides"):
        attend(v_pages=v[..., :16])
    with pytest.raises(ValueError, match="CUDA"):
        attend()
    qkv, cs, pos = torch.zeros(3, 8 * 64, dtype=torch.bfloat16), torch.zeros(9, 32, 2), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="scales"):
        kernels.paged_rope_kv(qkv, cs, pos, k, v, pos, 4, 2)
    with pytest.raises(ValueError, match="supported"):
        kernels.paged_rope_kv(qkv, cs, pos, k.to(torch.int8), v.to(torch.int8), pos, 4, 2, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.paged_kv_read(k, v, table, torch.tensor([0, 1, 2]), 2, k_scale=ks, v_scale=vs)
    w = torch.ones(64, dtype=torch.bfloat16)
    own = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)
    norm = lambda a, b: kernels.paged_norm_rope_kv(qkv, a, b, cs, pos, own, own.clone(), pos, 4, 2)  # noqa: E731
    for bad in (w.float(), w[:32], torch.ones(128, dtype=torch.bfloat16)[::2], w[None]):
        with pytest.raises(ValueError, match="q_norm and k_norm"):
            norm(bad, w)
        with pytest.raises(ValueError, match="q_norm and k_norm"):
            norm(w, bad)
    with pytest.raises(ValueError, match="CUDA"):
        norm(w, w)
