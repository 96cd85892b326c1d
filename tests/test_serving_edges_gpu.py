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
