"""Steps of a paged cache that bring no tokens, without a GPU (nothing is launched)."""

import pytest
import torch

from omniasr_b200.paged import PagedCache


@pytest.mark.parametrize("sequences", [0, 1, 3])
def test_steps_without_tokens(sequences):
    c = PagedCache(1, 4, 4, 2, 16, device="cpu")
    seqs = [c.add() for _ in range(sequences)]
    batch = c.extend(seqs, [0] * sequences)
    assert batch.tokens == 0 and batch.total == 0 and batch.table.shape == (sequences, 1)
    qkv, cs = torch.zeros(0, 8 * 16, dtype=torch.bfloat16), torch.zeros(8, 8, 2)
    for step in (c.decode, c.prefill):
        out = step(0, qkv, cs, batch, 4)
        assert out.shape == (0, 4, 16) and out.dtype == torch.bfloat16
    assert c.free_pages == 4
