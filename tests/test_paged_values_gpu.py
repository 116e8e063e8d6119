"""Attention over pages where the softmax is not an ordinary one.

Tolerances: see test_paged_gpu for the rounding of outputs, probabilities and sums."""

import pytest
import torch

from omniasr_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("heads,kv,dim,rows", [(8, 8, 128, 32), (16, 4, 128, 48), (16, 2, 64, 40), (32, 2, 128, 40), (8, 8, 512, 20), (8, 2, 256, 40)])
@pytest.mark.parametrize("nats", [11.0, 11.4, 11.8, 12.2, 12.5, 13.0])
def test_a_key_far_above_a_long_tail(heads, kv, dim, rows, nats):
    """8-bit pages, one key 11 to 13 nats above 32767 others that score alike, values with a common mean: each weight of the
    tail lies below the smallest step of the two e4m3 pieces (2^-13; the key's weight is 2^4 to 2^8), yet together they are
    a tenth of the sum and more. The units are long enough that few are cut.

    Beside the rounding of the output and of the weights' 8 significant bits (2^-8 (|o| + A), 2^-10 A), a weight's last piece
    is off by an error of mean zero within one step, a standard deviation of at most half of one: over n keys and a sum l >= 2^4
    that is sqrt(n) 2^-14 / l of a value; six of them (2.4e5 results, about 5e-4 of one expected past it)."""
    n, page = 32768, 128
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
