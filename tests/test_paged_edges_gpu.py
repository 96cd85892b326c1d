"""The paged cache's operators (GPU) where a call meets an edge: values that are not finite, caps far above
the scores, status bits across steps, one token's strides.  Bars as in test_paged_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch
from test_paged_gpu import attention_ref, check_attention, make

from m1moe_b200 import M1MoECudaError, PagedBatch, paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu


def test_a_status_bit_outlives_the_next_plan():
    """A bad page id in one step is still reported after the plan has been made again."""
    nh, nkv, hd, page = 8, 8, 128, 16
    cache, table, _ = make(nkv, hd, page, [1, 1], [40, 20], seed=31)
    good = table.clone()
    table[1, 1] = 10 ** 6
    batch = PagedBatch(cache, [1, 1], [40, 20], table, num_heads=nh)
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    paged_attention(cache, 0, batch, q)
    table.copy_(good)
    for _ in range(3):
        batch.update()
        paged_attention(cache, 0, batch, q)
    with pytest.raises(M1MoECudaError, match="0x2"):
        batch.check()
    batch.update()
    paged_attention(cache, 0, batch, q)
    batch.check()  # reported once


def test_a_new_batch_starts_without_status_bits():
    """Whatever its memory held before: batches made and dropped after raising a bit."""
    nh, nkv, hd, page = 8, 8, 128, 16
    cache, table, _ = make(nkv, hd, page, [1, 1], [40, 20], seed=32)
    bad = torch.full_like(table, 10 ** 6)
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    for _ in range(4):
        batch = PagedBatch(cache, [1, 1], [40, 20], bad, num_heads=nh)
        paged_attention(cache, 0, batch, q)
        del batch
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        for kw in ({}, {"stream": s}):
            batch = PagedBatch(cache, [1, 1], [40, 20], table, num_heads=nh, **kw)
            paged_attention(cache, 0, batch, q, **kw)
            batch.check(**kw)
            del batch


@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e8, 3e38])
@pytest.mark.parametrize("hd,q_lens,kv_lens", [(128, [1, 1, 1], [1, 700, 33]), (64, [2, 1], [90, 64]),
                                               (128, [70, 200], [300, 200]), (64, [130], [130])])
def test_caps_far_above_the_scores(hd, q_lens, kv_lens, cap):
    """cap tanh(s / cap) of scores between a ten-thousandth and a few times the cap: as the cap grows the
    result is the uncapped one.  Errors of tanh are relative (6e-7 at most), so scores of up to about 20 are
    off by about 1e-5, far inside the bar's 2^-11."""
    nh, nkv = 16, 4
    cache, table, dense = make(nkv, hd, 16, q_lens, kv_lens, seed=33)
    q = (3 * torch.randn((sum(q_lens), nh, hd), device="cuda")).bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    out = paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=torch.float32)
    batch.check()
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 1 / math.sqrt(hd), 0, cap)
    check_attention(out, ref, mag)
