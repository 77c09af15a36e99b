"""Batches that the allocator's kernels refuse while they run: the state stays
whole, however the warps of the one CTA come to see the error."""

import pytest
import torch

from agentkv_b200 import PoolConfig
from agentkv_b200.allocator import SlabAllocator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [33, 600, 2048])
def test_a_refused_dec_ref_batch_changes_nothing(n):
    """One id out of range, at every stretch of the batch: the record is
    written by the first warps to count, and the others go on with the same plan."""
    total = 2500
    a = SlabAllocator(PoolConfig(total_blocks=total, block_size=1, num_layers=1, num_kv_heads=1, head_dim=16,
                                 dtype="float16", device="cuda"))
    held = torch.tensor(a.alloc_many(n), dtype=torch.int32, device="cuda")
    a.check()
    refs = a._ref_counts.clone()
    for at in list(range(0, n, max(1, n // 40))) + [n - 1]:
        ids = held.clone()
        ids[at] = (total, -1, 2 ** 31 - 1)[at % 3]
        a.dec_ref_batch(ids)
        with pytest.raises(ValueError, match="out of range"):
            a.check()
        assert torch.equal(a._ref_counts, refs)
    a.dec_ref_batch(held)
    a.check()
    assert not a._ref_counts.any()
