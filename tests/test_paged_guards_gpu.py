"""Calls that the paged operators refuse before a launch (GPU)."""
from __future__ import annotations

import pytest
import torch

from m1moe_b200 import PagedBatch, PagedKVCache, paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu


def test_a_cache_of_fewer_pages_than_the_batchs_is_refused():
    make = lambda pages: PagedKVCache(num_layers=1, num_kv_heads=4, num_pages=pages, page_size=16)
    cache, small = make(8), make(6)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    batch = PagedBatch(cache, [1, 2], [60, 50], table, num_heads=8)
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros((3, 16 * 128), device="cuda")
    rope = rope_table(64, 128)
    with pytest.raises(ValueError, match="batch was made for"):
        paged_attention(small, 0, batch, q)
    with pytest.raises(ValueError, match="batch was made for"):
        paged_append(small, 0, batch, qkv, rope=rope)
    other = make(8)  # the same sizes: taken
    paged_append(other, 0, batch, qkv, rope=rope)
    paged_attention(other, 0, batch, q)
    batch.check()
