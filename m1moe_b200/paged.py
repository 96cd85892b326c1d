"""A paged key/value cache and its operators, for batches of sequences of different lengths.

Thin wrappers over the C ABI (include/m1moe_cuda.h, m1moe_cuda_paged_*); torch supplies
device memory and streams, every computation runs in libm1moe_cuda.so.

  PagedKVCache     the bf16 pools of every layer, [layers][pages][kv heads][page size][head dim]
  PagedBatch       one step's sequences: their new tokens, lengths and pages, and the plan that
                   every layer's calls share
  paged_append     per-head RMSNorm, rotary embedding and the store of the new keys and values
                   (InferenceEngine.swift:194-220, 521-548)
  paged_attention  causal attention over the pages (InferenceEngine.swift:349-399)
  rope_table       cosines and sines of every position, also scaled for long contexts

A batch's calls use its plan's partial results and so belong on one stream, in order.  They take
the cache that the batch was made for, or one with the same sizes on the same device.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .expert_ffn import _empty, _keep, dtype_code

_F32, _BF16 = torch.float32, torch.bfloat16
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream() without its wrapper: 0.1 of 3 us
_current_device = torch._C._cuda_getDevice


def _fn(name: str):
    """The entry point `name`, called with device `index` current (a null stream is that of the
    current device, whatever device the pointers are of) and its status checked."""
    f = None

    def call(index, *args):
        nonlocal f
        if f is None:
            f = getattr(_lib.lib(), name)
        if index == _current_device():
            st = f(*args)
        else:
            with torch.cuda.device(index):
                st = f(*args)
        if st:
            _lib.check(st, name)

    return call


_plan_call, _append_call = _fn("m1moe_cuda_paged_plan"), _fn("m1moe_cuda_paged_append")
_attention_call, _status_call = _fn("m1moe_cuda_paged_attention"), _fn("m1moe_cuda_paged_status")


class PagedKVCache:
    def __init__(self, *, num_layers: int, num_kv_heads: int, num_pages: int, page_size: int,
                 head_dim: int = 128, device: int = 0):
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        dev = torch.device("cuda", device)
        self._adopt(torch.zeros(shape, dtype=torch.bfloat16, device=dev),
                    torch.zeros(shape, dtype=torch.bfloat16, device=dev))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKVCache":
        """Pools that the caller owns: bf16 [layers][pages][kv heads][page size][head dim]."""
        self = cls.__new__(cls)
        self._adopt(k, v)
        return self

    def _adopt(self, k, v):
        if k.dim() != 5 or k.shape != v.shape:
            raise ValueError("k and v are [layers][pages][kv heads][page size][head dim]")
        for t in (k, v):
            if not t.is_cuda or t.dtype != torch.bfloat16 or not t.is_contiguous():
                raise ValueError("the pools are contiguous bfloat16 CUDA tensors")
        if k.device != v.device:
            raise ValueError("k and v are on different devices")
        self.k, self.v = k, v
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        self.device = k.device
        self._index = k.device.index
        self._layer_bytes = k[0].numel() * 2 if self.num_layers else 0
        self._k0, self._v0 = k.data_ptr(), v.data_ptr()

    def _ptrs(self, layer: int) -> tuple[int, int]:
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} out of range [0,{self.num_layers})")
        return self._k0 + layer * self._layer_bytes, self._v0 + layer * self._layer_bytes

    def _sizes(self):
        """What a batch's page ids and addresses are checked and formed by."""
        return self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self.device


class PagedBatch:
    """The sequences of one step.

    q_lens      new tokens of each sequence (host integers; 0 is allowed)
    kv_lens     all tokens of each sequence, the new ones included (host integers or an int32
                CUDA tensor, kept as `kv_lens`)
    page_table  int32 CUDA [sequences][most pages]; unused entries are never read
    window      positions a token sees, itself included (0: all before it)
    shared_prefix  positions at the start, whole pages, that all page tables share: attention
                   may then read them once for the batch; a hint that changes results by no
                more than rounding
    """

    def __init__(self, cache: PagedKVCache, q_lens, kv_lens, page_table: torch.Tensor, *, num_heads: int,
                 window: int = 0, shared_prefix: int = 0, stream=None):
        dev = cache.device
        q = [int(x) for x in (q_lens.tolist() if isinstance(q_lens, torch.Tensor) else q_lens)]
        if not q or min(q) < 0:
            raise ValueError("q_lens: at least one sequence, no negative length")
        if not isinstance(kv_lens, torch.Tensor):
            kv_lens = torch.tensor([int(x) for x in kv_lens], dtype=torch.int32, device=dev)
        for t, name, dim in ((kv_lens, "kv_lens", 1), (page_table, "page_table", 2)):
            if t.device != dev or t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError(f"{name}: a contiguous int32 tensor of {dim} dimension(s) on {dev}")
            if t.shape[0] != len(q):
                raise ValueError(f"{name} has {t.shape[0]} rows for {len(q)} sequences")
        cu = [0]
        for x in q:
            cu.append(cu[-1] + x)
        self.cache, self.page_table, self.kv_lens = cache, page_table, kv_lens
        self.num_seqs, self.total_q, self.max_q = len(q), cu[-1], max(q)
        self.num_heads = num_heads
        self.cfg = _lib.PagedCfg(num_heads, cache.num_kv_heads, cache.head_dim, cache.page_size, cache.num_pages,
                                 len(q), page_table.shape[1], cu[-1], max(q), window, shared_prefix)
        self._cfg = ctypes.addressof(self.cfg)
        with torch.cuda.device(dev):
            nbytes = _lib.lib().m1moe_cuda_paged_plan_bytes(self._cfg)
            if nbytes == 0:
                msg = _lib.lib().m1moe_cuda_last_error()
                raise ValueError(f"paged batch refused: {msg.decode() if msg else ''}")
        with torch.cuda.stream(stream):  # (None: the current one)
            self.cu_q = torch.tensor(cu, dtype=torch.int32, device=dev)
            # torch's allocations are 512-byte aligned; the plan's header starts without status bits
            self.plan = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            self.plan[:64].zero_()
        self._home = _raw_stream(dev.index) if stream is None else stream.cuda_stream
        _keep(stream if stream is not None else torch.cuda.current_stream(dev), kv_lens, page_table)
        self._plan, self._table = self.plan.data_ptr(), page_table.data_ptr()
        self._q_shape = (cu[-1], num_heads, cache.head_dim)
        self._qkv_shape = (cu[-1], (num_heads + 2 * cache.num_kv_heads) * cache.head_dim)
        self.update(stream=stream)

    def update(self, *, stream=None) -> None:
        """Make the plan again from `cu_q`, `kv_lens` and `page_table` as they are on the device
        now (for a next step with the same new tokens per sequence; capturable)."""
        st = self._use(stream)
        _plan_call(self.cache._index, self._cfg, self.cu_q.data_ptr(), self.kv_lens.data_ptr(), self._table,
                   self._plan, self.plan.numel(), st)

    def _made_for(self, cache: PagedKVCache) -> None:
        """Refuse a cache whose pools are not of the sizes that the plan goes by: the kernels would leave them."""
        if cache is not self.cache and cache._sizes() != self.cache._sizes():
            raise ValueError(f"the batch was made for a cache of (pages, kv heads, page size, head dim, device) "
                             f"{self.cache._sizes()}, not {cache._sizes()}")

    def check(self, *, stream=None) -> None:
        """Wait for the stream and raise if a kernel found a length, page or position out of range, in any
        step since the last check."""
        _status_call(self.cache._index, self._plan, self._use(stream))

    def _use(self, stream) -> int:
        st = _raw_stream(self.cache._index) if stream is None else stream.cuda_stream
        if st != self._home:  # keep the memory until this stream is done with it
            s = stream if stream is not None else torch.cuda.current_stream(self.cache.device)
            for t in (self.plan, self.cu_q, self.kv_lens, self.page_table):
                t.record_stream(s)
        return st


def paged_append(cache: PagedKVCache, layer: int, batch: PagedBatch, qkv: torch.Tensor, *, rope: torch.Tensor,
                 rope_pairs: bool = False, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                 eps: float = 1e-5, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Store the batch's new keys and values; returns the queries, bf16 [total_q][heads][head dim].

    qkv     f32 or bf16 [total_q][(heads + 2 kv heads) * head dim], rows q | k | v, which may lie
            further apart than their length
    rope    f32 [positions][rot/2][2] (rope_table); rot <= head dim elements of each head turn, i
            with i + rot/2 or, with rope_pairs, 2i with 2i + 1
    q_norm, k_norm  bf16 [head dim] RMSNorm weights of each head, or None
    """
    batch._made_for(cache)
    if qkv.shape != batch._qkv_shape:
        raise ValueError(f"qkv is {tuple(qkv.shape)}, expected {batch._qkv_shape}")
    dev = cache.device
    if qkv.device != dev or qkv.stride(1) != 1:
        raise ValueError("qkv: rows of contiguous elements on the cache's device")
    if rope.dim() != 3 or rope.dtype != _F32 or rope.shape[2] != 2 or rope.device != dev or not rope.is_contiguous():
        raise ValueError("rope: a contiguous float32 [positions][rot/2][2] tensor on the cache's device")
    qn = kn = 0
    if q_norm is not None:
        qn = _norm_ptr(q_norm, cache)
    if k_norm is not None:
        kn = _norm_ptr(k_norm, cache)
    k, v = cache._ptrs(layer)
    st = batch._use(stream)
    if out is None:
        out = _empty(batch._q_shape, _BF16, dev, stream)
    elif out.shape != batch._q_shape or out.dtype != _BF16 or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out: contiguous bfloat16 {batch._q_shape} on the cache's device")
    if batch.total_q == 0:
        return out
    _keep(stream, qkv, rope, q_norm, k_norm, out, cache.k, cache.v)
    positions, pairs, _ = rope.shape
    # one token's stride may be anything; the C side wants at least its length
    stride = qkv.stride(0) if batch.total_q > 1 else batch._qkv_shape[1]
    _append_call(cache._index, batch._cfg, batch._plan, batch._table, qkv.data_ptr(), dtype_code(qkv.dtype), stride,
                 qn, kn, eps, rope.data_ptr(), positions, 2 * pairs, 1 if rope_pairs else 0, k, v, out.data_ptr(), st)
    return out


def _norm_ptr(w: torch.Tensor, cache: PagedKVCache) -> int:
    if w.device != cache.device or w.dtype != _BF16 or w.shape != (cache.head_dim,) or not w.is_contiguous():
        raise ValueError(f"norm weights: contiguous bfloat16 [{cache.head_dim}] on the cache's device")
    return w.data_ptr()


def paged_attention(cache: PagedKVCache, layer: int, batch: PagedBatch, q: torch.Tensor, *,
                    scale: float | None = None, softcap: float = 0.0, out: torch.Tensor | None = None,
                    out_dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """Attention of the batch's new tokens (q bf16 [total_q][heads][head dim], tokens may lie
    further apart) over their sequences; scores are scale * q.k (default 1/sqrt(head dim)), capped
    as softcap * tanh(score / softcap) if softcap > 0."""
    batch._made_for(cache)
    if q.dtype != _BF16:
        raise TypeError(f"q must be bfloat16, got {q.dtype}")
    stride = _check_rows(q, "q", cache, batch)
    k, v = cache._ptrs(layer)
    st = batch._use(stream)
    if out is None:
        out = _empty(batch._q_shape, out_dtype, cache.device, stream)
        out_stride = batch._qkv_shape[1] - 2 * cache.num_kv_heads * cache.head_dim
    else:
        out_stride = _check_rows(out, "out", cache, batch)
    if batch.total_q == 0:
        return out
    _keep(stream, q, out, cache.k, cache.v)
    _attention_call(cache._index, batch._cfg, batch._plan, batch._table, q.data_ptr(), stride, k, v,
                    1.0 / math.sqrt(cache.head_dim) if scale is None else scale, softcap, out.data_ptr(),
                    dtype_code(out.dtype), out_stride, st)
    return out


def _check_rows(t: torch.Tensor, name: str, cache: PagedKVCache, batch: PagedBatch) -> int:
    """The token stride of t [total_q][heads][head dim], heads contiguous."""
    rows, inner, last = t.stride() if t.dim() == 3 else (0, 0, 0)
    if inner != cache.head_dim and batch.num_heads == 1:
        inner = cache.head_dim  # (one head's stride may be anything)
    if t.shape != batch._q_shape or t.device != cache.device or last != 1 or inner != cache.head_dim:
        raise ValueError(f"{name}: {batch._q_shape} with contiguous heads on the cache's device")
    # one token's stride may be anything; the C side wants at least its length
    return rows if batch.total_q > 1 else batch.num_heads * cache.head_dim


def rope_table(max_positions: int, rot_dim: int, *, theta: float = 10000.0, scaling: dict | None = None,
               device=None) -> torch.Tensor:
    """f32 [max_positions][rot_dim/2][2]: cos and sin of position * theta^(-2i/rot_dim), made in 64 bits.

    scaling, for contexts longer than the model was trained on (original = its trained length):
      {"type": "linear", "factor": f}  positions divided by f
      {"type": "ntk", "factor": f}     theta raised so that the slowest pair turns f times slower
      {"type": "yarn", "factor": f, "original": n, "beta_fast": 32, "beta_slow": 1}
          pairs that turn more than beta_fast times in n positions stay, those below beta_slow are
          divided by f, a ramp between; cosines and sines times 0.1 ln f + 1
    """
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be a positive even number")
    kind = (scaling or {}).get("type")
    f = float((scaling or {}).get("factor", 1.0))
    if kind not in (None, "linear", "ntk", "yarn") or f < 1.0:
        raise ValueError(f"unknown rope scaling {scaling}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if kind == "ntk":
        theta = theta * f ** (rot_dim / max(rot_dim - 2, 1))
    inv = theta ** (-i / rot_dim)
    gain = 1.0
    if kind == "linear":
        inv = inv / f
    elif kind == "yarn":
        n = float(scaling["original"])
        lo, hi = float(scaling.get("beta_slow", 1.0)), float(scaling.get("beta_fast", 32.0))
        # linear in the pair's number between the numbers at which it turns hi and lo times, which may
        # lie before the first pair or beyond the last
        at = lambda t: rot_dim * math.log(n / (2 * math.pi * t)) / (2 * math.log(theta))
        a, b = math.floor(at(hi)), math.ceil(at(lo))
        ramp = ((i / 2 - a) / max(b - a, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / f * ramp
        gain = 0.1 * math.log(f) + 1.0
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * inv
    return (torch.stack((angle.cos(), angle.sin()), dim=-1) * gain).float().to(device if device is not None else "cuda")
