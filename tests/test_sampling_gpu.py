"""The sampler (GPU) against its definition in 64 bits.

The token is a whole number, so it has to be the definition's; the kernel's
weights are fp32 exponentials (relative error below 2^-20 with their
argument's rounding at |x| <= 25, then cut to 2^-36 of the largest), so where u
or top_p lies within DELTA of a boundary either neighbour is right:
DELTA = 2e-5 covers 25 * 2^-24 + 2^-22 with 150001 tokens cut by 2^-36 each.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from m1moe_b200 import M1MoECudaError, sample

pytestmark = pytest.mark.gpu
DELTA = 2e-5


def token_ref(x, u, temp, k, p, mp):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1
    if not temp > 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temp))
    w = e.copy()
    if k > 0:
        w[k:] = 0
    if p < 1:
        need = p * w.sum()
        w[1:][np.cumsum(w)[:-1] >= need] = 0
    w[e < mp] = 0
    by = np.zeros_like(w)
    by[order] = w
    run = np.cumsum(by)
    return int(np.searchsorted(run, min(max(u, 0.0), 1 - 2.0 ** -24) * run[-1], side="right"))


def allowed(x, u, temp, k, p, mp):
    s = set()
    for du in (-DELTA, 0, DELTA):
        for dp in (-DELTA, 0, DELTA) if 0 < p < 1 else (0,):
            for dm in (-DELTA, 0, DELTA) if 0 < mp < 1 else (0,):
                s.add(token_ref(x, min(max(u + du, 0), 1), temp, k, p * (1 + dp), mp * (1 + dm)))
    return s


def check(logits, u, temp, k, p, mp):
    """Per-row settings as tensors."""
    t = lambda a, d=torch.float32: torch.tensor(np.asarray(a), dtype=d, device="cuda")
    got = sample(logits, t(u), temperature=t(temp), top_k=t(k, torch.int32), top_p=t(p), min_p=t(mp))
    again = sample(logits, t(u), temperature=t(temp), top_k=t(k, torch.int32), top_p=t(p), min_p=t(mp))
    assert got.dtype == torch.int32 and torch.equal(got, again)
    x = logits.float().cpu().numpy()
    f = np.float32
    for r, tok in enumerate(got.tolist()):
        ok = allowed(x[r], float(f(u[r])), float(f(temp[r])), int(k[r]), float(f(p[r])), float(f(mp[r])))
        assert tok in ok, (r, tok, ok, temp[r], k[r], p[r], mp[r])
    return got


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (2, 33), (1, 50304), (5, 32000), (80, 8193),
                                        (2, 150001), (1, 400000), (200, 515), (160, 60001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_settings_vs_definition(rows, vocab, dtype):
    rng = np.random.default_rng(rows * 7 + vocab)
    x = rng.normal(0, 2.5, size=(rows, vocab)).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, vocab, size=min(vocab, 30))] += 6
    logits = torch.from_numpy(x).cuda().to(dtype)
    pick = lambda *a: rng.choice(a, size=rows)
    check(logits, rng.random(rows).astype(np.float32), pick(0.0, 0.5, 0.8, 1.0, 1.7), pick(0, 1, 2, 40, 1000),
          pick(0.0, 0.5, 0.9, 0.99, 1.0), pick(0.0, 0.0, 0.05, 0.3))


@pytest.mark.parametrize("rows,vocab", [(40, 3000), (4, 50304)])
def test_each_filter_alone(rows, vocab):
    rng = np.random.default_rng(2)
    logits = torch.from_numpy(rng.normal(0, 3, size=(rows, vocab)).astype(np.float32)).cuda()
    u = rng.random(rows).astype(np.float32)
    one, zero = np.ones(rows), np.zeros(rows)
    for k in (0, 1, 7, vocab - 1, vocab, vocab + 5, -3):
        check(logits, u, one, np.full(rows, k), one, zero)
    for p in (0.0, 1e-6, 0.3, 0.97, 0.999999, 1.0, 1.5):
        check(logits, u, one, zero, np.full(rows, p), zero)
    for mp in (1e-4, 0.2, 1.0):
        check(logits, u, one, zero, one, np.full(rows, mp))
    for t in (1e-30, 1e-3, 0.1, 5.0, 1e30, math.inf):
        check(logits, u, np.full(rows, t), zero, one, zero)


def test_every_token_is_reached_in_proportion():
    """u on a fine grid gives each token its probability's share, to the grid's step."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1.5, size=97).astype(np.float32)
    n = 1 << 14
    u = (torch.arange(n, device="cuda") + 0.5) / n
    logits = torch.from_numpy(x).cuda()[None].expand(n, 97)  # rows 0 elements apart
    got = sample(logits.contiguous(), u, temperature=0.9)
    share = torch.bincount(got.long(), minlength=97).double().cpu().numpy() / n
    p = np.exp(x.astype(np.float64) / np.float32(0.9))
    assert np.all(np.abs(share - p / p.sum()) <= 2.0 / n)
    assert torch.all(got[1:] >= got[:-1])  # by index


@pytest.mark.parametrize("vocab", [64, 20000, 70001])
def test_ties_go_to_the_lower_index(vocab):
    u = torch.tensor([0.0, 0.5, 0.999999], device="cuda")
    flat = torch.zeros((3, vocab), device="cuda")
    assert sample(flat, u, temperature=0.0).tolist() == [0, 0, 0]
    # of equal tokens top_k keeps the first ones by index
    got = sample(flat, u, top_k=10).tolist()
    assert got == [0, 5, 9]
    got = sample(flat, u, top_p=0.25)
    kept = math.ceil(vocab * 0.25)
    assert got.tolist() == [0, int(kept * 0.5), kept - 1]
    # equal tokens behind a larger one: 1 + 4 of the ties
    flat[:, vocab // 2] = 3.0
    got = sample(flat, torch.tensor([0.0, 0.0, 0.999999], device="cuda"), top_k=5, temperature=1e6).tolist()
    assert got == [0, 0, vocab // 2]
    # +0 and -0 are equal
    flat = torch.tensor([[-1.0, -0.0, 0.0, -2.0]], device="cuda")
    assert sample(flat, u[:1], temperature=0.0).tolist() == [1]
    assert sample(flat, u[:1], top_k=1).tolist() == [1]


def test_infinities_and_nan():
    inf, nan = math.inf, math.nan
    u = torch.tensor([0.6], device="cuda")
    row = lambda *a: torch.tensor([a], device="cuda")
    assert sample(row(-inf, -inf, -inf), u).tolist() == [-1]
    assert sample(row(nan, -inf, nan), u).tolist() == [-1]
    assert sample(row(nan, 1.0, nan), u).tolist() == [1]
    assert sample(row(-inf, 0.0, -inf, 0.0), u).tolist() == [3]
    assert sample(row(1.0, inf, 5.0, inf), u).tolist() == [3]
    assert sample(row(1.0, inf, 5.0, inf), u, top_k=1).tolist() == [1]
    assert sample(row(1.0, inf, 5.0, inf), u, top_p=0.5).tolist() == [1]
    assert sample(row(-3.4e38, -3.4e38), u).tolist() == [1]
    assert sample(row(3.4e38, -3.4e38), u).tolist() == [0]
    # the type's lowest value as a mask
    low = torch.finfo(torch.bfloat16).min
    x = torch.full((1, 5000), low, dtype=torch.bfloat16, device="cuda")
    x[0, 4321] = -2.0
    assert sample(x, u, top_k=50, top_p=0.9).tolist() == [4321]
    # settings that are no numbers never leave a row without a token
    x = torch.randn((1, 3000), device="cuda")
    bad = torch.tensor([nan], device="cuda")
    for kw in ({"temperature": bad}, {"top_p": bad}, {"min_p": bad}, {"min_p": torch.tensor([7.0], device="cuda")}):
        assert 0 <= sample(x, u, **kw).item() < 3000
    assert 0 <= sample(x, bad).item() < 3000
    assert 0 <= sample(x, torch.tensor([1.0], device="cuda")).item() < 3000


def test_cut_among_values_near_zero():
    """A cut inside a cluster of values around 0, where floats are densest."""
    rng = np.random.default_rng(8)
    x = np.concatenate([rng.normal(0, 1e-20, 4000), [1e-38, -1e-38, 1e-45, -1e-45], rng.normal(0, 1e-3, 500)])
    x = x.astype(np.float32)[None].repeat(6, 0)
    logits = torch.from_numpy(x).cuda()
    u = np.linspace(0.05, 0.95, 6).astype(np.float32)
    for k in (3, 700, 2500):
        # all weights are 1 to 2^-9: the k kept ones are exact, by rank
        got = check(logits, u, np.ones(6), np.full(6, k), np.ones(6), np.zeros(6))
        order = np.argsort(-x[0], kind="stable")[:k]
        assert set(got.tolist()) <= set(order.tolist())


def test_rows_apart_and_output_and_scalars():
    rng = np.random.default_rng(9)
    wide = torch.from_numpy(rng.normal(0, 3, size=(6, 1500)).astype(np.float32)).cuda()
    x = wide[:, 1:1002]
    u = torch.rand(6, device="cuda")
    out = torch.full((6,), -7, dtype=torch.int32, device="cuda")
    got = sample(x, u, temperature=0.7, top_k=50, top_p=0.9, out=out)
    assert got is out
    ref = sample(x.contiguous(), u, temperature=torch.full((6,), 0.7, device="cuda"),
                 top_k=torch.full((6,), 50, dtype=torch.int32, device="cuda"),
                 top_p=torch.full((6,), 0.9, device="cuda"))
    assert torch.equal(out, ref)
    # a row does not depend on the others
    for r in range(6):
        assert sample(x[r:r + 1], u[r:r + 1], temperature=0.7, top_k=50, top_p=0.9).item() == out[r].item()
    assert sample(torch.empty((0, 10), device="cuda"), torch.empty(0, device="cuda")).shape == (0,)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = sample(x, u, temperature=0.7, top_k=50, top_p=0.9, stream=s)
    s.synchronize()
    assert torch.equal(other, out)


def test_refusals():
    x, u = torch.zeros((2, 8), device="cuda"), torch.zeros(2, device="cuda")
    for kw in ({"temperature": -1.0}, {"temperature": math.nan}, {"top_p": -0.1}, {"min_p": 1.5}, {"min_p": -0.5}):
        with pytest.raises(M1MoECudaError):
            sample(x, u, **kw)
    with pytest.raises(M1MoECudaError):
        sample(torch.zeros((1, (1 << 20) + 1), device="cuda"), u[:1])
    with pytest.raises(ValueError):
        sample(x, 0.5)
    with pytest.raises(ValueError):
        sample(x, u[:1])
    with pytest.raises(ValueError):
        sample(x, u, top_k=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        sample(x.t(), torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError):
        sample(x, u, out=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        sample(x.half(), u)
