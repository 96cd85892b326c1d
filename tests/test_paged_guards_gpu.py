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


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30, 900])
@pytest.mark.parametrize("q_lens,kv_lens", [([4, 1, 4], [2, 40, 4]), ([400, 1, 300, 131], [100, 700, 300, 1])])
def test_a_window_beyond_every_position_hides_nothing(q_lens, kv_lens, window):
    """Also for sequences shorter than their new tokens, whose first tokens lie before position 0."""
    nh, nkv, hd, page = 4, 2, 128, 16
    cache = PagedKVCache(num_layers=1, num_kv_heads=nkv, num_pages=160, page_size=page)
    g = torch.Generator(device="cuda").manual_seed(41)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    table = torch.randperm(160, generator=g, device="cuda")[:40 * len(q_lens)] if len(q_lens) == 3 else None
    if table is None:
        table = torch.arange(160, device="cuda")
    table = table.int().view(len(q_lens), -1)
    table = torch.nn.functional.pad(table, (0, 50 - table.shape[1]), value=0).contiguous()
    q = torch.randn((sum(q_lens), nh, hd), generator=g, device="cuda").bfloat16()
    outs = []
    for w in (0, window):
        batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=w)
        outs.append(paged_attention(cache, 0, batch, q))
        batch.check()
    assert outs[0].any() and torch.equal(outs[0], outs[1])
