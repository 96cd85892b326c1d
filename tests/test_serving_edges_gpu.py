"""The whole step and the generation loop (GPU) where a call meets an edge: the model's own rotation base, errors
of the MoE block, streams, top-2 routing.  The bar is test_serving_gpu.py's."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from test_serving_gpu import BAR, logits_of

from m1moe_b200 import M1MoECudaError, MoEBlock, PagedBatch, PagedKVCache, rope_table, synth
from m1moe_b200.dense import DenseModel
from m1moe_b200.serving import generate

pytestmark = pytest.mark.gpu


def model(seed, nh, nkv, qk_norm, *, top_k=8, layers=2, vocab=1000, h=256, theta=1e4, max_batch=8):
    dm = DenseModel(hidden_dim=h, num_heads=nh, num_kv_heads=nkv, num_layers=layers, vocab_size=vocab,
                    qk_norm=qk_norm, rope_theta=theta, max_batch=max_batch, max_seq=256)
    w = synth.dense_weights(seed, h=h, nh=nh, nkv=nkv, hd=128, layers=layers, vocab=vocab, qk_norm=qk_norm)
    dm.load_all(w)
    blk = MoEBlock(hidden_dim=h, intermediate_dim=128, num_experts=8, top_k=top_k, num_layers=layers,
                   norm_topk_prob=not qk_norm, max_batch=8)
    for L in range(layers):
        blk.load_expert_layer(L, synth.layer_image(seed + 100 + L, 8, h, 128, 64))
        blk.load_router(L, synth.router_weights(seed + 200 + L, 8, h))
    return dm, blk, w


@pytest.mark.parametrize("theta", [1e6, 300.0])
def test_generate_rotates_by_the_models_own_base(theta):
    dm, blk, _ = model(51, 2, 2, True, theta=theta)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, size=n).tolist() for n in (60, 41, 90)]
    out = generate(dm, blk, prompts, max_new_tokens=4, page_size=16, temperature=0.0).tolist()
    for p, new in zip(prompts, out):
        for i, t in enumerate(new):
            ref = logits_of(dm, blk, p + new[:i])
            assert ref[t] >= ref.max() - 2 * BAR * ref.abs().max(), i
    # a base given by name still counts: the same numbers, the same tokens
    again = generate(dm, blk, prompts, max_new_tokens=1, page_size=16, temperature=0.0, rope_theta=theta).tolist()
    assert [x[:1] for x in out] == again
    dm.close()
    blk.close()


def test_generate_reports_the_moe_blocks_errors():
    """Activations beyond the range of the prompt's tensor-core operands raise, as in MoEBlock.synchronize."""
    dm, blk, _ = model(52, 2, 2, True)
    huge = torch.full((256,), 1e7).bfloat16()
    dm.load("post_norm", huge, 0)
    with pytest.raises(M1MoECudaError):
        generate(dm, blk, [list(range(30))], max_new_tokens=1, page_size=16, temperature=0.0)
    dm.close()
    blk.close()


def step_parts(dm, nkv, lens, nh, stream=None):
    cache = PagedKVCache(num_layers=dm.num_layers, num_kv_heads=nkv, num_pages=sum(-(-n // 16) for n in lens), page_size=16)
    table = torch.full((len(lens), max(-(-n // 16) for n in lens)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        x = -(-n // 16)
        table[b, :x] = torch.arange(at, at + x, dtype=torch.int32)
        at += x
    return cache, table.cuda()


def test_outputs_belong_to_the_stream_that_fills_them(monkeypatch):
    """Memory for an output comes from the pool of the stream the call runs on: the current stream's
    pool may hold a block that queued work still uses."""
    dm, blk, _ = model(53, 2, 2, True)
    cache, table = step_parts(dm, 2, [3, 4], 2)
    s = torch.cuda.Stream()
    toks = torch.arange(7, dtype=torch.int32, device="cuda")
    rope = rope_table(16, 128)
    batch = PagedBatch(cache, [3, 4], [3, 4], table, num_heads=2)
    torch.cuda.synchronize()
    made, empty = [], torch.empty

    def record(*a, **kw):
        made.append(torch.cuda.current_stream().cuda_stream)
        return empty(*a, **kw)

    monkeypatch.setattr(torch, "empty", record)
    lg = dm.paged_step(blk, cache, batch, toks, rope=rope, stream=s)
    assert made and set(made) == {s.cuda_stream}
    made.clear()
    dm.reset()
    dm.prefill(blk, toks, stream=s)
    dm.step(blk, toks[:1], stream=s)
    dm.lm_head(torch.zeros((1, 256), device="cuda"), stream=s)
    dm.attention(0, torch.zeros((1, 6 * 128), device="cuda"), stream=s)
    x = torch.zeros((2, 256), device="cuda")
    blk.forward(0, x, return_topk=True, stream=s)
    blk.prefill(0, x, return_topk=True, stream=s)
    blk.route(0, x, stream=s)
    assert made and set(made) == {s.cuda_stream}
    monkeypatch.undo()
    s.synchronize()
    assert lg.isfinite().all()
    dm.close()
    blk.close()


def test_top_2_routing_matches_the_contiguous_model():
    """Two of eight experts a token.  Where two experts are nearly equal a rounding may rightly swap them, so
    the prompts compared are those whose contiguous logits stay within the bar when the output projections
    are perturbed by up to 2^-7 of each element, at random and four times: twice the size of the paged
    path's own roundings (2^-8) of what enters them."""
    dm, blk, w = model(54, 4, 2, False, top_k=2)
    rng = np.random.default_rng(4)
    seqs = [rng.integers(0, 1000, size=n).tolist() for n in list(range(1, 25)) + [40, 60, 33, 50]]
    cache, table = step_parts(dm, 2, [len(s) for s in seqs], 4)
    rope = rope_table(128, 128)
    as_ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = PagedBatch(cache, [len(s) for s in seqs], [len(s) for s in seqs], table, num_heads=4)
    lg = dm.paged_step(blk, cache, batch, as_ints([t for s in seqs for t in s]), rope=rope).clone()
    # the same last tokens again as single-token steps of up to eight sequences, after the others
    one = torch.zeros_like(lg)
    for i in range(0, len(seqs), 8):
        part = seqs[i:i + 8]
        c, t = step_parts(dm, 2, [len(s) for s in part], 4)
        if any(len(s) > 1 for s in part):
            b = PagedBatch(c, [len(s) - 1 for s in part], [len(s) - 1 for s in part], t, num_heads=4)
            dm.paged_step(blk, c, b, as_ints([x for s in part for x in s[:-1]]), rope=rope)
        b = PagedBatch(c, [1] * len(part), [len(s) for s in part], t, num_heads=4)
        one[i:i + 8] = dm.paged_step(blk, c, b, as_ints([s[-1] for s in part]), rope=rope)
        b.check()
    dm.synchronize()
    refs = [logits_of(dm, blk, s) for s in seqs]
    steady = [True] * len(seqs)
    g = torch.Generator().manual_seed(6)
    wo = [torch.from_numpy(np.asarray(x)).view(torch.bfloat16).float() for x in w["wo"]]
    for _ in range(4):
        for L, x in enumerate(wo):
            noise = 1 + 2.0 ** -7 * (2 * torch.rand(x.shape, generator=g) - 1)
            dm.load("wo", (x * noise).bfloat16().view(torch.int16), L)
        for b, s in enumerate(seqs):
            moved = (logits_of(dm, blk, s) - refs[b]).abs().max()
            steady[b] = steady[b] and bool(moved <= BAR * refs[b].abs().max())
    assert sum(steady) >= len(seqs) // 4, sum(steady)
    for b, ok in enumerate(steady):
        if ok:
            for got in (lg[b], one[b]):
                assert (got - refs[b]).abs().max() <= BAR * refs[b].abs().max(), (b, len(seqs[b]))
    dm.close()
    blk.close()
