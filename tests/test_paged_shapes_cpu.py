"""Shapes whose sizes pass the integers that the host counts in: needs no GPU."""
from __future__ import annotations

import pytest
from test_paged_cpu import lib, plan_bytes  # noqa: F401  (lib is a fixture)


@pytest.mark.parametrize("huge", [
    # 2^30 pages of 2^24 heads and 1024 rows: 2^64 rows, 0 in 64 bits
    dict(num_heads=2 ** 24, num_kv_heads=2 ** 24, page_size=1024, num_pages=2 ** 30, num_seqs=1, total_q=1,
         max_pages_per_seq=1),
    dict(num_heads=2 ** 27, num_kv_heads=2 ** 27, page_size=16, num_pages=2 ** 30 + 1, num_seqs=1, total_q=1,
         max_pages_per_seq=1),
    dict(num_heads=2 ** 30, num_kv_heads=2 ** 30, page_size=1024, num_pages=2 ** 30, num_seqs=1, total_q=1,
         max_pages_per_seq=1),
])
def test_sizes_whose_product_passes_64_bits_are_refused(lib, huge):
    assert plan_bytes(lib, **huge) == 0
    assert b"31 bits" in lib.m1moe_cuda_last_error()
