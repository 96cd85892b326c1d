"""Sampled generation for a batch of prompts over a paged cache: the serving loop in small.

`generate` admits all prompts at once (one ragged step; a prefix that the prompts share is
computed and cached once), then takes one token per sequence a step -- append, attention
(the shared prefix read once for the batch), MoE layers, logits, sampling -- with everything
of a step on the GPU.  The reference generates one sequence token by token and samples on the
CPU (bench/main.swift:139-160, InferenceEngine.swift:124-156, 550-575).
"""
from __future__ import annotations

import torch

from .paged import PagedBatch, PagedKVCache, rope_table
from .sampling import sample


def shared_prefix(prompts: list[list[int]], page_size: int) -> int:
    """Positions, in whole pages, that all prompts share and none consists of alone."""
    if len(prompts) < 2:
        return 0
    n = min(len(p) for p in prompts) - 1
    for i in range(n):
        if any(p[i] != prompts[0][i] for p in prompts):
            n = i
            break
    return max(n, 0) // page_size * page_size


def generate(dense, moe, prompts: list[list[int]], *, max_new_tokens: int, rope: torch.Tensor | None = None,
             rope_theta: float | None = None, page_size: int = 64, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             generator: torch.Generator | None = None) -> torch.Tensor:
    """int32 tokens [prompts][max_new_tokens] (CUDA).  dense: DenseModel, moe: its MoEBlock;
    rope: the rotation table, by default that of rope_theta, by default the model's own;
    the settings are sampling.sample's."""
    if not prompts or any(not p for p in prompts) or max_new_tokens < 1:
        raise ValueError("at least one prompt, none of them empty, and at least one new token")
    dev = torch.device("cuda", dense.device)
    n = len(prompts)
    last = [len(p) + max_new_tokens for p in prompts]
    shared = shared_prefix(prompts, page_size)
    sp = shared // page_size
    need = [-(-t // page_size) - sp for t in last]
    cache = PagedKVCache(num_layers=dense.num_layers, num_kv_heads=dense.num_kv_heads, num_pages=sp + sum(need),
                         page_size=page_size, head_dim=dense.head_dim, device=dense.device)
    table = torch.full((n, sp + max(need)), -1, dtype=torch.int32)
    at = sp
    for b, x in enumerate(need):
        table[b, :sp] = torch.arange(sp, dtype=torch.int32)
        table[b, sp:sp + x] = torch.arange(at, at + x, dtype=torch.int32)
        at += x
    table = table.to(dev)
    if rope is None:
        theta = dense.cfg.rope_theta if rope_theta is None else rope_theta
        rope = rope_table(max(last), dense.head_dim, theta=theta, device=dev)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    if shared:
        one = PagedBatch(cache, [shared], [shared], table[:1].contiguous(), num_heads=dense.num_heads)
        dense.paged_step(moe, cache, one, ints(prompts[0][:shared]), rope=rope)
        one.check()
    rest = [p[shared:] for p in prompts]
    batch = PagedBatch(cache, [len(p) for p in rest], [len(p) for p in prompts], table, num_heads=dense.num_heads)
    logits = dense.paged_step(moe, cache, batch, ints([t for p in rest for t in p]), rope=rope)
    batch.check()
    out = torch.empty((max_new_tokens, n), dtype=torch.int32, device=dev)
    settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    lens = ints([len(p) for p in prompts])
    batch = None
    for i in range(max_new_tokens):
        sample(logits, torch.rand(n, generator=generator, device=dev), out=out[i], **settings)
        if i + 1 == max_new_tokens:
            break
        lens += 1
        if batch is None:
            batch = PagedBatch(cache, [1] * n, lens, table, num_heads=dense.num_heads, shared_prefix=shared)
        else:
            batch.update()
        dense.paged_step(moe, cache, batch, out[i], rope=rope, logits=logits)
    if batch is not None:
        batch.check()
    dense.synchronize()
    moe.synchronize()  # (each reports its own kernels' errors)
    return out.t().contiguous()
