"""Token sampling from logits: temperature, top-k, top-p and min-p, one uniform number per row.

Thin wrapper over m1moe_cuda_sample (include/m1moe_cuda.h), which defines the result exactly
(whole-number weights, ties to the lower index); replaces the CPU sampling of
InferenceEngine.swift:550-575.
"""
from __future__ import annotations

import torch

from .expert_ffn import _empty, _keep, dtype_code
from .paged import _fn, _raw_stream

_sample_call = _fn("m1moe_cuda_sample")
_F32, _I32 = torch.float32, torch.int32


def _setting(t, name: str, dtype: torch.dtype, rows: int, dev) -> tuple[int, float]:
    """(pointer, 0) of a tensor [rows], or (0, value) of a number."""
    if not isinstance(t, torch.Tensor):
        return 0, t
    if t.dtype != dtype or t.shape != (rows,) or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor [{rows}] on {dev}")
    return t.data_ptr(), 0


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """int32 tokens [rows] from logits [rows][vocab] (f32 or bf16, rows may lie further apart) and
    u f32 [rows] in [0, 1).  Each setting is a number or a CUDA tensor [rows] (f32; top_k int32).
    temperature 0: the largest logit; top_k <= 0, top_p >= 1 and min_p 0 leave that filter off; a
    row of -inf gives -1."""
    if logits.dim() != 2 or not logits.is_cuda or (logits.numel() and logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: a CUDA tensor [rows][vocab] of contiguous rows")
    rows, vocab = logits.shape
    dev = logits.device
    if not isinstance(u, torch.Tensor):
        raise ValueError("u is a tensor of one uniform number per row")
    pu, _ = _setting(u, "u", _F32, rows, dev)
    pt, vt = _setting(temperature, "temperature", _F32, rows, dev)
    pk, vk = _setting(top_k, "top_k", _I32, rows, dev)
    pp, vp = _setting(top_p, "top_p", _F32, rows, dev)
    pm, vm = _setting(min_p, "min_p", _F32, rows, dev)
    st = _raw_stream(dev.index) if stream is None else stream.cuda_stream
    if out is None:
        out = _empty((rows,), _I32, dev, stream)
    elif out.device != dev or out.dtype != _I32 or out.shape != (rows,) or not out.is_contiguous():
        raise ValueError(f"out: a contiguous int32 tensor [{rows}] on {dev}")
    _keep(stream, logits, u, temperature, top_k, top_p, min_p, out)
    # one row's stride may be anything; the C side wants at least the row's length
    stride = logits.stride(0) if rows > 1 else max(logits.stride(0), vocab)
    _sample_call(dev.index, logits.data_ptr(), dtype_code(logits.dtype), stride, rows, vocab, pu, pt, vt, pk, vk, pp, vp,
                 pm, vm, out.data_ptr(), st)
    return out
