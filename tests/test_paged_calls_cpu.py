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


@pytest.fixture
def devices(monkeypatch):
    """Two devices, 0 the current one: the list of devices that the entry points ran on."""
    state, ran = {"now": 0}, []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["now"] = state["now"], self.index

        def __exit__(self, *exc):
            state["now"] = self.before

    class Lib:
        def __getattr__(self, name):
            return lambda *a: ran.append((name, state["now"])) or 0

    monkeypatch.setattr(paged, "_current_device", lambda: state["now"])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "lib", Lib)
    for name in ("plan", "append", "attention", "status"):
        monkeypatch.setattr(paged, f"_{name}_call", paged._fn(f"m1moe_cuda_paged_{name}"))
    return ran


@pytest.mark.parametrize("index", [0, 1])
def test_calls_run_on_the_caches_device(index, devices):
    """Raw stream 0 is the default stream of whichever device is current: the call makes the tensors'
    device current, and only then."""
    batch = fake_batch(fake_cache())
    batch.cache._index = index
    batch.cu_q = batch.kv_lens = batch.plan = torch.zeros(1)
    append(batch.cache, batch)
    attend(batch.cache, batch)
    batch.update()
    batch.check()
    assert devices == [(f"m1moe_cuda_paged_{x}", index) for x in ("append", "attention", "plan", "status")]
    assert paged._current_device() == 0


@pytest.mark.parametrize("index", [0, 1])
def test_sampling_runs_on_the_logits_device(index, devices, monkeypatch):
    from m1moe_b200 import sampling

    class Logits:  # a CUDA tensor's face
        is_cuda, dtype, shape = True, torch.float32, (2, 5)
        device = torch.device("cuda", index)

        def dim(self):
            return 2

        def numel(self):
            return 10

        def stride(self, i):
            return (5, 1)[i]

        def data_ptr(self):
            return 64

    monkeypatch.setattr(sampling, "_setting", lambda t, *a: (0, 0))
    monkeypatch.setattr(sampling, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(sampling, "_empty", lambda *a: torch.zeros(2, dtype=torch.int32))
    monkeypatch.setattr(sampling, "_sample_call", paged._fn("m1moe_cuda_sample"))
    sampling.sample(Logits(), torch.zeros(2))
    assert devices == [("m1moe_cuda_sample", index)]
    assert paged._current_device() == 0


@pytest.mark.parametrize("on", ["cache", "tokens", "rope", "logits"])
def test_a_whole_step_over_two_devices_is_refused(on, calls):
    """The model's kernels run on its own device and would be given another one's pointers."""
    from m1moe_b200.dense import DenseModel

    class Face:  # a tensor's face
        def __init__(self, shape, dtype, device):
            self.shape, self.dtype, self.device, self.is_cuda = shape, dtype, torch.device("cuda", device), True

        def dim(self):
            return len(self.shape)

        def is_contiguous(self):
            return True

    at = lambda name: 1 if on == name else 0
    dm = DenseModel.__new__(DenseModel)
    dm.num_layers, dm.vocab_size, dm.device = 2, 100, 0
    cache = fake_cache(device=torch.device("cuda", at("cache")))
    if on == "cache":  # all but the model
        at = lambda name: 1
    with pytest.raises(ValueError, match="device|model on"):
        dm.paged_step(None, cache, fake_batch(cache), Face((3,), torch.int32, at("tokens")),
                      rope=Face((64, HD // 2, 2), torch.float32, at("rope")),
                      logits=Face((3, 100), torch.float32, at("logits")))
