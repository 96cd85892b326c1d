"""Calls on another stream than the current one (GPU): the memory of what they read stays until they have run.

Each test keeps the other stream busy, queues a call there, drops its inputs and fills memory of the same
size on the current stream: the allocator must not hand out the inputs' blocks before the call has run."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from test_paged_gpu import make
from test_serving_gpu import model

from m1moe_b200 import PagedBatch, PagedKVCache, paged_append, paged_attention, rope_table, sample

pytestmark = pytest.mark.gpu
BUSY = 20_000_000  # cycles: about ten milliseconds


def late(s, call):
    """call(s) behind other work of s."""
    torch.cuda.synchronize()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(BUSY)
    return call(s)


def overwrite(*shapes):
    """Memory of these shapes and types, as the current stream's pool gives it, filled with ones."""
    return [torch.ones(shape, dtype=dtype, device="cuda") for shape, dtype in shapes for _ in range(12)]


def test_inputs_of_append_and_attention():
    nh, nkv, hd, page = 16, 4, 128, 16
    cache, table, _ = make(nkv, hd, page, [30, 1], [60, 90], seed=71)
    rope = rope_table(100, hd)
    batch = PagedBatch(cache, [30, 1], [60, 90], table, num_heads=nh)
    g = torch.Generator(device="cuda").manual_seed(72)
    qkv0 = torch.randn((31, (nh + 2 * nkv) * hd), generator=g, device="cuda").bfloat16()
    q0 = paged_append(cache, 0, batch, qkv0, rope=rope)
    want = paged_attention(cache, 0, batch, q0)
    s = torch.cuda.Stream()
    qkv = qkv0.clone()
    q = late(s, lambda s: paged_append(cache, 0, batch, qkv, rope=rope, stream=s))
    del qkv
    junk = overwrite((qkv0.shape, qkv0.dtype))
    s.synchronize()
    assert torch.equal(q, q0)
    del junk
    q = q0.clone()
    out = late(s, lambda s: paged_attention(cache, 0, batch, q, stream=s))
    del q
    junk = overwrite((q0.shape, q0.dtype))
    s.synchronize()
    assert torch.equal(out, want)
    del junk


def test_inputs_of_sampling():
    g = torch.Generator(device="cuda").manual_seed(73)
    x0, u0 = 3 * torch.randn((40, 30000), generator=g, device="cuda"), torch.rand(40, generator=g, device="cuda")
    k0 = torch.full((40,), 50, dtype=torch.int32, device="cuda")
    want = sample(x0, u0, top_k=k0, temperature=0.9)
    s = torch.cuda.Stream()
    x, u, k = x0.clone(), u0.clone(), k0.clone()
    got = late(s, lambda s: sample(x, u, top_k=k, temperature=0.9, stream=s))
    del x, u, k
    junk = overwrite((x0.shape, x0.dtype), (u0.shape, u0.dtype), (k0.shape, k0.dtype))
    s.synchronize()
    assert torch.equal(got, want)
    del junk


def test_inputs_of_a_whole_step():
    dm, blk = model(74, 4, 2, False)
    cache = PagedKVCache(num_layers=2, num_kv_heads=2, num_pages=12, page_size=16)
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    batch = PagedBatch(cache, [50, 9], [50, 9], table, num_heads=4)
    toks0 = torch.from_numpy(np.random.default_rng(7).integers(2, 1000, size=59).astype(np.int32)).cuda()
    rope = rope_table(64, 128)
    want = dm.paged_step(blk, cache, batch, toks0, rope=rope)
    s = torch.cuda.Stream()
    toks, table2 = toks0.clone(), rope.clone()
    lg = late(s, lambda s: dm.paged_step(blk, cache, batch, toks, rope=table2, stream=s))
    del toks, table2
    junk = overwrite((toks0.shape, toks0.dtype), (rope.shape, rope.dtype))
    s.synchronize()
    assert (lg - want).abs().max() <= 1e-3 * want.abs().max()
    del junk
    dm.close()
    blk.close()


def test_a_batch_made_on_another_stream():
    """Its page table and lengths were allocated on the current one."""
    nh, nkv, hd, page = 16, 4, 128, 16
    cache, table0, _ = make(nkv, hd, page, [1, 1], [60, 90], seed=75)
    lens0 = torch.tensor([60, 90], dtype=torch.int32, device="cuda")
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    want = paged_attention(cache, 0, PagedBatch(cache, [1, 1], lens0, table0, num_heads=nh), q)
    for given in (False, True):
        s = torch.cuda.Stream()
        table, lens = table0.clone(), lens0.clone()

        def call(s):
            if given:
                batch = PagedBatch(cache, [1, 1], lens, table, num_heads=nh, stream=s)
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    torch.cuda._sleep(BUSY)
                batch.update(stream=s)
                return paged_attention(cache, 0, batch, q, stream=s)
            with torch.cuda.stream(s):
                batch = PagedBatch(cache, [1, 1], lens, table, num_heads=nh)
                torch.cuda._sleep(BUSY)
                batch.update()
                return paged_attention(cache, 0, batch, q)

        out = late(s, call)
        del table, lens
        junk = overwrite((table0.shape, table0.dtype), (lens0.shape, lens0.dtype))
        s.synchronize()
        assert torch.equal(out, want)
        del junk
