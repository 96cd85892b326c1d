"""Captured steps (GPU) beside larger calls of the same contexts: a graph's buffers stay its own.

The replayed step and the eager one run the same kernels; the MoE block sums with atomics, so the last
bits may differ: the bar is 1e-3 of the largest logit."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from test_serving_gpu import model

from m1moe_b200 import M1MoECudaError, PagedBatch, PagedKVCache, rope_table

pytestmark = pytest.mark.gpu


def captured(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()  # the kernels and buffers of this size
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fn()
    return graph


def batch_of(cache, q_lens, first_page, nh):
    table = torch.arange(first_page, first_page + 20 * len(q_lens), dtype=torch.int32, device="cuda").view(len(q_lens), 20)
    return PagedBatch(cache, q_lens, q_lens, table, num_heads=nh)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [2, 1, 2], [10, 1, 30]])  # the decode kernels twice, the prompt ones
def test_a_captured_step_survives_larger_calls(q_lens):
    dm, blk = model(61, 4, 2, False)
    rng = np.random.default_rng(5)
    ints = lambda n: torch.tensor(rng.integers(0, 1000, size=n), dtype=torch.int32, device="cuda")
    cache = PagedKVCache(num_layers=2, num_kv_heads=2, num_pages=400, page_size=16)
    rope = rope_table(320, 128)
    small = batch_of(cache, q_lens, 0, 4)
    toks = ints(sum(q_lens))
    lg = torch.zeros((3, 1000), device="cuda")

    def step():
        small.update()
        dm.paged_step(blk, cache, small, toks, rope=rope, logits=lg)

    graph = captured(step)
    for grow in ([100], [300, 200], [7] * 16):  # more tokens; more sequences
        large = batch_of(cache, grow, 60, 4)
        t = ints(sum(grow))
        first = dm.paged_step(blk, cache, large, t, rope=rope)
        toks.copy_(ints(sum(q_lens)))
        step()
        want = lg.clone()
        lg.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (lg - want).abs().max() <= 1e-3 * want.abs().max()
        again = dm.paged_step(blk, cache, large, t, rope=rope)  # and the graph leaves the larger call alone
        assert (again - first).abs().max() <= 1e-3 * first.abs().max()
    small.check()
    dm.synchronize()
    blk.synchronize()
    dm.close()
    blk.close()


def test_a_captured_prefill_survives_larger_calls():
    dm, blk = model(62, 2, 2, True)
    rng = np.random.default_rng(6)
    ints = lambda n: torch.tensor(rng.integers(0, 1000, size=n), dtype=torch.int32, device="cuda")
    toks, lg = ints(20), torch.zeros(1000, device="cuda")
    graph = captured(lambda: dm.prefill(blk, toks, logits=lg))
    for n in (90, 200):
        dm.reset()
        dm.prefill(blk, ints(n))
        dm.reset()
        dm.prefill(blk, toks, logits=lg)
        dm.synchronize()
        want = lg.clone()
        lg.zero_()
        dm.reset()
        torch.cuda.synchronize()
        graph.replay()
        dm.synchronize()
        assert (lg - want).abs().max() <= 1e-3 * want.abs().max()
    dm.close()
    blk.close()


def test_growth_while_capturing_is_refused():
    dm, blk = model(63, 2, 2, True)
    cache = PagedKVCache(num_layers=2, num_kv_heads=2, num_pages=40, page_size=16)
    rope = rope_table(64, 128)
    small, large = batch_of(cache, [3], 0, 2), batch_of(cache, [30], 20, 2)
    toks = torch.zeros(30, dtype=torch.int32, device="cuda")
    lg = torch.zeros((1, 1000), device="cuda")
    dm.paged_step(blk, cache, small, toks[:3], rope=rope, logits=lg)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(M1MoECudaError, match="captured"):
            dm.paged_step(blk, cache, large, toks, rope=rope, logits=lg)
        dm.paged_step(blk, cache, small, toks[:3], rope=rope, logits=lg)
    graph.replay()
    dm.synchronize()
    dm.paged_step(blk, cache, large, toks, rope=rope, logits=lg)
    dm.synchronize()
    assert lg.isfinite().all()
    dm.close()
    blk.close()
