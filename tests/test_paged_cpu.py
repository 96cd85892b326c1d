"""Host-side parts of the paged cache that need no GPU: shapes that are refused, rotation tables,
the prefix that prompts share."""
from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from m1moe_b200 import build
    build.build()
    from m1moe_b200 import _lib
    return _lib.lib()


def plan_bytes(lib, **kw):
    from m1moe_b200._lib import PagedCfg
    shape = dict(num_heads=32, num_kv_heads=8, head_dim=128, page_size=64, num_pages=1000, num_seqs=4,
                 max_pages_per_seq=100, total_q=4, max_q=1, window=0, shared_prefix=0)
    shape.update(kw)
    cfg = PagedCfg(*[shape[n] for n, _ in PagedCfg._fields_])
    return lib.m1moe_cuda_paged_plan_bytes(ctypes.addressof(cfg))


def test_plan_bytes_of_good_shapes(lib):
    base = plan_bytes(lib)
    assert base > 0
    assert plan_bytes(lib, head_dim=64, page_size=16) > 0
    assert plan_bytes(lib, total_q=4000, max_q=1000) > base  # 256-row items: larger partials
    assert plan_bytes(lib, total_q=0, max_q=0) > 0
    assert plan_bytes(lib, num_seqs=40, total_q=40, shared_prefix=640) > plan_bytes(lib, num_seqs=40, total_q=40)


@pytest.mark.parametrize("bad,why", [
    (dict(num_heads=30), b"multiple"), (dict(num_heads=136), b"at most 16"), (dict(num_kv_heads=0), b"positive"),
    (dict(head_dim=96), b"64 or 128"), (dict(page_size=24), b"power of two"), (dict(page_size=8), b"power of two"),
    (dict(page_size=2048), b"power of two"), (dict(num_pages=0), b"positive"), (dict(num_seqs=0), b"positive"),
    (dict(total_q=-1), b">= 0"), (dict(max_q=5), b"does not fit"), (dict(total_q=5), b"does not fit"),
    (dict(window=-1), b"window"), (dict(shared_prefix=65), b"multiple of the page size"),
    (dict(shared_prefix=6464), b"longer"), (dict(num_pages=2 ** 24), b"31 bits"),
    (dict(max_pages_per_seq=2 ** 26), b"31 bits"),
    (dict(num_seqs=2 ** 20, total_q=2 ** 20, max_pages_per_seq=2 ** 14), b"31 bits"),
])
def test_shapes_that_are_refused(lib, bad, why):
    assert plan_bytes(lib, **bad) == 0
    assert why in lib.m1moe_cuda_last_error()


def test_null_pointers_are_refused(lib):
    assert lib.m1moe_cuda_paged_plan_bytes(None) == 0
    assert lib.m1moe_cuda_paged_status(None, None) == 1
    assert lib.m1moe_cuda_sample(None, 0, 10, 1, 10, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None) == 1
    assert lib.m1moe_cuda_sample(None, 2, 10, 1, 10, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None) == 1
    assert lib.m1moe_cuda_sample(None, 0, 10, 0, 10, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None) == 0


def test_rope_table_rows_are_rotations():
    from m1moe_b200.paged import rope_table
    t = rope_table(100, 64, theta=500.0, device="cpu")
    assert t.shape == (100, 32, 2) and t.dtype == torch.float32
    assert torch.allclose((t.double() ** 2).sum(-1), torch.ones(100, 32, dtype=torch.float64), atol=1e-6)
    assert torch.equal(t[0], torch.tensor([[1.0, 0.0]]).expand(32, 2))
    # turning by a and then by b is turning by a + b
    z = torch.view_as_complex(t.double().contiguous())
    assert torch.allclose(z[17] * z[40], z[57], atol=1e-6)


def test_shared_prefix_of_prompts():
    from m1moe_b200.serving import shared_prefix
    a = list(range(100))
    assert shared_prefix([a], 16) == 0
    assert shared_prefix([a, a], 16) == 96
    assert shared_prefix([a, a[:40] + [7]], 16) == 32
    assert shared_prefix([a, [5] + a], 16) == 0
    assert shared_prefix([a[:16], a], 16) == 0  # the shorter prompt keeps a token of its own
