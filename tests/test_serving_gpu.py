"""A whole model over the paged cache (GPU) against the same model over its contiguous cache.

Both run the same weights; the paged step's attention takes bf16 queries, weights and outputs
(relative rounding 2^-8 each) where the contiguous one keeps f32.  The attention output enters
the residual beside terms of its own size, so the logits may move by about 3 * 2^-8 of their own
size at most: |difference| <= 1.2e-2 of the largest logit is the bar (a wrong row, position or
page moves them by their whole size).  Every token goes to all eight experts: with a top-2
router a rounding that swaps two near-equal experts moves the logits by far more, rightly."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from m1moe_b200 import MoEBlock, PagedBatch, PagedKVCache, rope_table, synth
from m1moe_b200.dense import DenseModel
from m1moe_b200.serving import generate, shared_prefix

pytestmark = pytest.mark.gpu
BAR = 1.2e-2


def model(seed, nh, nkv, qk_norm, B=8, layers=2, vocab=1000, h=256, max_seq=256):
    dm = DenseModel(hidden_dim=h, num_heads=nh, num_kv_heads=nkv, num_layers=layers, vocab_size=vocab,
                    qk_norm=qk_norm, rope_theta=1e4, max_batch=B, max_seq=max_seq)
    dm.load_all(synth.dense_weights(seed, h=h, nh=nh, nkv=nkv, hd=128, layers=layers, vocab=vocab, qk_norm=qk_norm))
    blk = MoEBlock(hidden_dim=h, intermediate_dim=128, num_experts=8, top_k=8, num_layers=layers,
                   norm_topk_prob=not qk_norm, max_batch=B)
    for L in range(layers):
        blk.load_expert_layer(L, synth.layer_image(seed + 100 + L, 8, h, 128, 64))
        blk.load_router(L, synth.router_weights(seed + 200 + L, 8, h))
    return dm, blk


def logits_of(dm, blk, tokens):
    dm.reset()
    lg = torch.empty((dm.vocab_size,), dtype=torch.float32, device="cuda")
    dm.prefill(blk, torch.tensor(tokens, dtype=torch.int32, device="cuda"), logits=lg)
    dm.synchronize()
    return lg


@pytest.mark.parametrize("nh,nkv,qk_norm", [(2, 2, True), (4, 2, False)])
def test_ragged_steps_match_the_contiguous_model(nh, nkv, qk_norm):
    dm, blk = model(11, nh, nkv, qk_norm)
    rng = np.random.default_rng(0)
    seqs = [rng.integers(0, 1000, size=n).tolist() for n in (70, 5, 33, 1, 64)]
    page = 16
    cache = PagedKVCache(num_layers=2, num_kv_heads=nkv, num_pages=30, page_size=page)
    table = torch.full((5, 8), -1, dtype=torch.int32)
    ids = rng.permutation(30)[:25].reshape(5, 5)
    table[:, :5] = torch.from_numpy(ids.astype(np.int32))
    table = table.cuda()
    rope = rope_table(128, 128)
    done = [0] * 5
    # prompts in chunks: many tokens (the prefill kernels), then few (the decode ones), one idle
    for q in ([60, 3, 30, 1, 64], [9, 0, 2, 0, 0], [1, 2, 1, 0, 0]):
        step = [s[d:d + n] for s, d, n in zip(seqs, done, q)]
        done = [d + len(x) for d, x in zip(done, step)]
        batch = PagedBatch(cache, [len(x) for x in step], done, table, num_heads=nh)
        toks = torch.tensor([t for x in step for t in x], dtype=torch.int32, device="cuda")
        lg = dm.paged_step(blk, cache, batch, toks, rope=rope)
        batch.check()
        for b, x in enumerate(step):
            if x:
                ref = logits_of(dm, blk, seqs[b][:done[b]])
                assert (lg[b] - ref).abs().max() <= BAR * ref.abs().max(), (q, b)
    assert done == [70, 5, 33, 1, 64]
    dm.close()
    blk.close()


def test_many_sequences_take_the_batched_head():
    dm, blk = model(21, 4, 2, False)
    rng = np.random.default_rng(1)
    seqs = [rng.integers(0, 1000, size=n).tolist() for n in range(1, 13)]
    cache = PagedKVCache(num_layers=2, num_kv_heads=2, num_pages=12, page_size=16)
    table = torch.arange(12, dtype=torch.int32, device="cuda")[:, None].contiguous()
    batch = PagedBatch(cache, [len(s) for s in seqs], [len(s) for s in seqs], table, num_heads=4)
    toks = torch.tensor([t for s in seqs for t in s], dtype=torch.int32, device="cuda")
    lg = dm.paged_step(blk, cache, batch, toks, rope=rope_table(16, 128))
    for b, s in enumerate(seqs):
        ref = logits_of(dm, blk, s)
        assert (lg[b] - ref).abs().max() <= BAR * ref.abs().max(), b
    dm.close()
    blk.close()


def test_generate_greedy_and_sampled():
    dm, blk = model(31, 2, 2, True)
    rng = np.random.default_rng(2)
    head = rng.integers(0, 1000, size=40).tolist()
    prompts = [head + rng.integers(0, 1000, size=n).tolist() for n in (3, 17, 1, 30)]
    assert shared_prefix(prompts, 16) == 32 and shared_prefix(prompts[:1], 16) == 0
    assert shared_prefix([head, head], 8) == 32  # one token at least is each prompt's own
    out = generate(dm, blk, prompts, max_new_tokens=6, page_size=16, temperature=0.0).tolist()
    for p, new in zip(prompts, out):
        for i, t in enumerate(new):  # each token is the largest logit, to the bar
            ref = logits_of(dm, blk, p + new[:i])
            assert ref[t] >= ref.max() - 2 * BAR * ref.abs().max(), i
    g = torch.Generator(device="cuda").manual_seed(5)
    a = generate(dm, blk, prompts, max_new_tokens=9, page_size=16, temperature=0.8, top_k=50, top_p=0.95, generator=g)
    g.manual_seed(5)
    b = generate(dm, blk, prompts, max_new_tokens=9, page_size=16, temperature=0.8, top_k=50, top_p=0.95, generator=g)
    assert a.shape == (4, 9) and int(a.min()) >= 0 and int(a.max()) < 1000
    # (the MoE block sums with atomics, so the last bits of logits may differ from run to run:
    # the first token, from the same prompts, is all that is compared)
    assert torch.equal(a[:, 0], b[:, 0])
    dm.close()
    blk.close()


def test_refusals():
    dm, blk = model(41, 2, 2, True)
    cache = PagedKVCache(num_layers=2, num_kv_heads=2, num_pages=4, page_size=16)
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    batch = PagedBatch(cache, [2], [2], table, num_heads=2)
    toks = torch.zeros(2, dtype=torch.int32, device="cuda")
    rope = rope_table(32, 128)
    with pytest.raises(ValueError):
        dm.paged_step(blk, cache, batch, toks[:1], rope=rope)
    with pytest.raises(ValueError):
        dm.paged_step(blk, cache, batch, toks, rope=rope.double())
    with pytest.raises(ValueError):
        dm.paged_step(blk, PagedKVCache(num_layers=1, num_kv_heads=2, num_pages=4, page_size=16), batch, toks, rope=rope)
    with pytest.raises(ValueError):
        generate(dm, blk, [[1], []], max_new_tokens=2)
    with pytest.raises(RuntimeError):  # four heads: not this model's batch
        dm.paged_step(blk, cache, PagedBatch(cache, [2], [2], table, num_heads=4), toks, rope=rope)
    dm.close()
    blk.close()
