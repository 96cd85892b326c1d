"""What the paged calls check and pass on before anything is launched: needs no GPU.  The C entry points are
stand-ins that record their arguments."""
from __future__ import annotations

import pytest
import torch

from m1moe_b200 import _lib, paged

HEADS, KV, HD = 4, 2, 128


def fake_cache(pages=10, kv=KV, page=16, hd=HD, layers=2, device=torch.device("cpu")):
    """A PagedKVCache's fields without its checks (the pools are host tensors)."""
    c = paged.PagedKVCache.__new__(paged.PagedKVCache)
    shape = (layers, pages, kv, page, hd)
    c.k, c.v = torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(shape, dtype=torch.bfloat16)
    c.num_layers, c.num_pages, c.num_kv_heads, c.page_size, c.head_dim = shape
    c.device, c._index = device, 0
    c._layer_bytes = c.k[0].numel() * 2
    c._k0, c._v0 = c.k.data_ptr(), c.v.data_ptr()
    return c


def fake_batch(cache, tokens=3):
    b = paged.PagedBatch.__new__(paged.PagedBatch)
    b.cache, b.num_heads, b.total_q, b.num_seqs = cache, HEADS, tokens, tokens
    b._q_shape = (tokens, HEADS, HD)
    b._qkv_shape = (tokens, (HEADS + 2 * KV) * HD)
    b._cfg = b._plan = b._table = b._home = 0
    b._use = lambda stream: 0
    return b


@pytest.fixture
def calls(monkeypatch):
    """The calls of the C entry points, as (name, arguments)."""
    made = []
    for name in ("_plan_call", "_append_call", "_attention_call", "_status_call"):
        monkeypatch.setattr(paged, name, lambda *a, name=name: made.append((name, a)))
    return made


def append(cache, batch):
    x = torch.zeros(batch._qkv_shape, dtype=torch.bfloat16)
    return paged.paged_append(cache, 0, batch, x, rope=torch.zeros((64, HD // 2, 2)))


def attend(cache, batch):
    return paged.paged_attention(cache, 0, batch, torch.zeros(batch._q_shape, dtype=torch.bfloat16))


def step(cache, batch):
    from m1moe_b200.dense import DenseModel
    dm = DenseModel.__new__(DenseModel)
    dm.num_layers, dm.vocab_size = 2, 100
    return dm.paged_step(None, cache, batch, torch.zeros(batch.total_q, dtype=torch.int32),
                         rope=torch.zeros((64, HD // 2, 2)))


@pytest.mark.parametrize("call", [append, attend, step])
@pytest.mark.parametrize("other", [dict(pages=9), dict(page=32), dict(pages=5, page=32), dict(kv=1), dict(hd=64),
                                   dict(device=torch.device("meta"))])
def test_a_batch_of_another_cache_is_refused(call, other, calls):
    """The kernels check page ids and form addresses by the batch's sizes: with a smaller pool behind them
    they would leave it."""
    batch = fake_batch(fake_cache())
    with pytest.raises(ValueError, match="batch was made for"):
        call(fake_cache(**other), batch)
    assert not calls


@pytest.mark.parametrize("call", [append, attend])
def test_a_cache_of_the_same_sizes_is_accepted(call, calls):
    """Two caches of equal sizes (a draft model's pools, a copy) may share a batch."""
    batch = fake_batch(fake_cache())
    call(batch.cache, batch)
    call(fake_cache(layers=7), batch)
    assert len(calls) == 2
