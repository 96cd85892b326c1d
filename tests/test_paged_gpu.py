"""The paged cache's append and attention (GPU) against plain 64-bit formulas.

Bars, derived before the first run.  bf16 rounds with relative error at most
2^-8 (8 significant bits).  append: v is rounded once, so it is equal to the
rounded input; q and k are one rounding of fp32 arithmetic whose own error
is below 2^-18 of the pair's magnitude (a 128-term sum of squares, a square
root and four products of relative error 2^-24 each).  attention:
  |out - ref| <= 2^-8 |ref|                     the output's rounding (bf16)
               + (2^-8 + 2^-11) sum_p w |v| / l   the weights' rounding, and the
                                                scores' fp32 errors (a 128-term
                                                dot product of |q.k| <= ~100:
                                                100 * 128 * 2^-24 < 2^-10 of a
                                                weight at the very worst)
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from m1moe_b200 import M1MoECudaError, PagedBatch, PagedKVCache, paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -8


def make(nkv, hd, page, q_lens, kv_lens, *, seed=0, spare=3, junk=-1, layers=1, share=0, fill=None):
    """A cache with the sequences' pages in random order, NaN in every row that belongs to no
    position; returns it with its page table and dense [t][nkv][hd] copies of each sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-t // page) for t in kv_lens]
    sp = share // page
    total = sp + sum(max(0, n - sp) for n in need) + spare
    k = torch.full((layers, total, nkv, page, hd), math.nan, dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    table = torch.full((len(need), max(max(need), 1)), junk, dtype=torch.int32)
    at = sp
    dense = []
    for b, n in enumerate(need):
        ids = order[:min(n, sp)] + order[at:at + max(0, n - sp)]
        at += max(0, n - sp)
        table[b, :n] = torch.tensor(ids, dtype=torch.int32)
        if n == 0:
            dense.append((torch.zeros((0, nkv, hd), device="cuda"),) * 2)
            continue
        idx = torch.tensor(ids, device="cuda")
        pos = torch.arange(kv_lens[b], device="cuda")
        for pool in (k, v):
            x = torch.randn((layers, kv_lens[b], nkv, hd), generator=g, device="cuda").bfloat16()
            old = pool[:, idx[pos // page], :, pos % page].permute(1, 0, 2, 3)
            x = torch.where(old.isnan(), x, old)  # a shared page keeps its first owner's rows
            pool[:, idx[pos // page], :, pos % page] = x.permute(1, 0, 2, 3)
        dense.append(tuple(pool[0, idx[pos // page], :, pos % page] for pool in (k, v)))
    return PagedKVCache.from_tensors(k, v), table.cuda(), dense


def attention_ref(q, dense, q_lens, kv_lens, nkv, scale, window=0, cap=0.0):
    """(ref, sum of w |v|) in 64 bits."""
    ref = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(ref)
    at, group = 0, q.shape[1] // nkv
    for (k, v), a, t in zip(dense, q_lens, kv_lens):
        k, v = k.double(), v.double()
        for i in range(0, a, 256):
            n = min(256, a - i)
            pos = torch.arange(t - a + i, t - a + i + n, device="cuda")
            see = torch.arange(t, device="cuda")[None] <= pos[:, None]
            if window:
                see &= torch.arange(t, device="cuda")[None] > pos[:, None] - window
            x = q[at + i:at + i + n].double().view(n, nkv, group, -1)
            s = torch.einsum("nhgd,thd->nhgt", x, k) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            s = s.masked_fill(~see[:, None, None], -math.inf)
            m = s.amax(-1, keepdim=True) if t else torch.zeros((n, nkv, group, 1), device="cuda")
            w = torch.exp(s - torch.where(m.isinf(), 0.0, m))
            l = w.sum(-1, keepdim=True)
            w = w / torch.where(l == 0, 1.0, l)
            ref[at + i:at + i + n] = torch.einsum("nhgt,thd->nhgd", w, v).reshape(n, -1, q.shape[2])
            mag[at + i:at + i + n] = torch.einsum("nhgt,thd->nhgd", w, v.abs()).reshape(n, -1, q.shape[2])
        at += a
    return ref, mag


def check_attention(out, ref, mag):
    bound = (U16 + 2.0 ** -11) * mag + 1e-30
    if out.dtype == torch.bfloat16:
        bound = bound + U16 * ref.abs()
    bad = ~((out.double() - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((out.double() - ref).abs().nan_to_num(9).max()))


CASES = [
    # nh, nkv, hd, page, q_lens, kv_lens, window, cap
    (16, 16, 128, 16, [1], [2048], 0, 0.0),
    (16, 16, 128, 16, [1], [1], 0, 0.0),
    (32, 8, 128, 64, [1] * 9, [1, 15, 16, 17, 63, 64, 65, 129, 5000], 0, 0.0),
    (32, 8, 64, 32, [1] * 5, [7, 31, 33, 400, 1025], 0, 30.0),
    (16, 1, 128, 128, [1, 1, 1], [127, 128, 4097], 100, 0.0),
    (24, 8, 128, 1024, [1] * 6, [1, 1023, 1024, 1025, 2049, 300], 1, 0.0),
    (8, 4, 64, 16, [1, 1, 1], [0, 40, 0], 0, 0.0),          # idle slots
    (8, 4, 128, 16, [0, 1, 0, 2], [33, 40, 0, 1], 0, 0.0),   # no new tokens; fewer positions than tokens
    (16, 16, 128, 32, [5, 1, 16], [5, 900, 77], 0, 0.0),      # short runs of new tokens
    (32, 8, 128, 64, [4, 3], [513, 4], 0, 20.0),
    (16, 16, 128, 16, [130, 1, 257], [130, 3000, 700], 0, 0.0),
    (32, 8, 128, 64, [300, 64, 33], [300, 64, 2000], 0, 0.0),
    (32, 8, 64, 128, [500, 7], [1500, 7], 0, 0.0),
    (24, 8, 128, 16, [171, 86], [400, 86], 0, 50.0),
    (16, 16, 128, 32, [700, 100, 1], [900, 2200, 800], 64, 0.0),
    (16, 1, 64, 16, [33, 17, 1], [33, 1000, 129], 37, 15.0),
    (16, 2, 128, 64, [1000, 0, 20], [1000, 50, 12], 0, 0.0),
    (4, 4, 128, 16, [2000], [2000], 300, 0.0),
]


@pytest.mark.parametrize("nh,nkv,hd,page,q_lens,kv_lens,window,cap", CASES)
def test_attention_vs_formula(nh, nkv, hd, page, q_lens, kv_lens, window, cap):
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=nh + hd + sum(kv_lens))
    g = torch.Generator(device="cuda").manual_seed(1)
    q = (2 * torch.randn((sum(q_lens), nh, hd), generator=g, device="cuda")).bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=window)
    out = paged_attention(cache, 0, batch, q, softcap=cap)
    batch.check()
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 1 / math.sqrt(hd), window, cap)
    check_attention(out, ref, mag)
    again = paged_attention(cache, 0, batch, q, softcap=cap)
    assert torch.equal(out, again)  # the same every time


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [700, 33, 2]), ([40, 1, 300], [40, 500, 310])])
def test_attention_strides_layer_scale_and_f32_output(q_lens, kv_lens):
    nh, nkv, hd, page = 32, 8, 128, 32
    cache, table, _ = make(nkv, hd, page, q_lens, kv_lens, layers=3, seed=4)
    n = sum(q_lens)
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn((n, nh * hd + 72), generator=g, device="cuda").bfloat16()
    q = wide[:, :nh * hd].unflatten(1, (nh, hd))
    outw = torch.full((n, nh * hd + 40), 7.0, device="cuda")
    out = outw[:, :nh * hd].unflatten(1, (nh, hd))
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    got = paged_attention(cache, 2, batch, q, scale=0.05, out=out)
    batch.check()
    assert got is out and torch.all(outw[:, nh * hd:] == 7.0)
    dense = []
    for b, t in enumerate(kv_lens):
        pos = torch.arange(t, device="cuda")
        idx = table[b].long()[pos // page]
        dense.append((cache.k[2][idx, :, pos % page], cache.v[2][idx, :, pos % page]))
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 0.05)
    check_attention(out, ref, mag)


def test_large_scores_and_equal_scores():
    """Scores of several hundred (one weight is 1, the rest vanish) and all-equal ones (the mean)."""
    nh = nkv = 4
    q_lens, kv_lens = [1, 70], [100, 200]
    cache, table, dense = make(nkv, 128, 16, q_lens, kv_lens, seed=6)
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    q = torch.zeros((71, nh, 128), dtype=torch.bfloat16, device="cuda")
    out = paged_attention(cache, 0, batch, q)
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 128 ** -0.5)
    check_attention(out, ref, mag)
    # powers of two: the products are exact in fp32 and so are the scores
    q = (64.0 * torch.randint(-1, 2, q.shape, device="cuda")).bfloat16()
    for pool in (cache.k,):
        pool.copy_(torch.where(pool.isnan(), pool, pool.sign() * 2.0))
    dense = [(d[0].sign() * 2.0, d[1]) for d in dense]
    out = paged_attention(cache, 0, batch, q, scale=0.25)
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 0.25)
    check_attention(out, ref, mag)


@pytest.mark.parametrize("q_len", [1, 40])
def test_pool_beyond_32_bit_offsets(q_len):
    """Pages whose element offset passes 2^31 and byte offset 2^32."""
    nkv, hd, page = 8, 128, 64
    pages = (2 ** 31) // (nkv * hd * page) + 40
    k = torch.zeros((1, pages, nkv, page, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    cache = PagedKVCache.from_tensors(k, v)
    kv = 300
    table = torch.arange(pages - 1, pages - 6, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn((kv, (16 + 2 * nkv) * hd), generator=g, device="cuda").bfloat16()
    rope = rope_table(kv, hd)
    fill = PagedBatch(cache, [kv], [kv], table, num_heads=16)
    q = paged_append(cache, 0, fill, qkv, rope=rope)
    fill.check()
    pos = torch.arange(kv, device="cuda")
    idx = table[0].long()[pos // page]
    dense = [(k[0][idx, :, pos % page], v[0][idx, :, pos % page])]
    assert torch.equal(dense[0][1], qkv[:, 24 * hd:].view(kv, nkv, hd))
    batch = PagedBatch(cache, [q_len], [kv], table, num_heads=16)
    out = paged_attention(cache, 0, batch, q[kv - q_len:])
    ref, mag = attention_ref(q[kv - q_len:], dense, [q_len], [kv], nkv, hd ** -0.5)
    check_attention(out, ref, mag)


# ------------------------------------------------------------------ append --
def append_ref(qkv, nh, nkv, hd, pos, rope, pairs, qn, kn, eps):
    x = qkv.double().view(-1, nh + 2 * nkv, hd)
    r = rope.double()[pos]
    half = rope.shape[1]

    def one(h, w):
        if w is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
        a, b = (h[..., 0:2 * half:2], h[..., 1:2 * half:2]) if pairs else (h[..., :half], h[..., half:2 * half])
        c, s = r[:, None, :, 0], r[:, None, :, 1]
        y, mag = h.clone(), h.abs()
        ya, yb, m = a * c - b * s, b * c + a * s, a.abs() + b.abs()
        if pairs:
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = ya, yb
            mag[..., 0:2 * half:2], mag[..., 1:2 * half:2] = m, m
        else:
            y[..., :half], y[..., half:2 * half] = ya, yb
            mag[..., :half], mag[..., half:2 * half] = m, m
        return y, mag

    return one(x[:, :nh], qn), one(x[:, nh:nh + nkv], kn), qkv.view(-1, nh + 2 * nkv, hd)[:, nh + nkv:].bfloat16()


def check_rounded(got, ref, mag):
    assert torch.all((got.double() - ref).abs() <= U16 * ref.abs() + 2.0 ** -18 * mag + 1e-30)


@pytest.mark.parametrize("nh,nkv,hd,page,q_lens,kv_lens", [
    (16, 16, 128, 16, [1], [2048]),
    (32, 8, 128, 64, [1] * 7, [1, 64, 65, 3000, 2, 0, 17]),
    (24, 8, 64, 32, [70, 0, 5, 1], [70, 9, 100, 33]),
    (16, 1, 128, 128, [3, 300], [2, 1000]),
    (4, 4, 64, 1024, [1025], [1500]),
])
@pytest.mark.parametrize("dtype,norm,rot,pairs", [
    (torch.float32, True, "all", False), (torch.bfloat16, False, "all", True), (torch.bfloat16, True, "half", False),
    (torch.float32, False, "half", True), (torch.float32, True, 16, False), (torch.float32, True, 48, True)])
def test_append_vs_formula(nh, nkv, hd, page, q_lens, kv_lens, dtype, norm, rot, pairs):
    rot = {"all": hd, "half": hd // 2}.get(rot, rot)
    cache, table, _ = make(nkv, hd, page, q_lens, kv_lens, seed=9)
    before = [cache.k.clone(), cache.v.clone()]
    n, width = sum(q_lens), (nh + 2 * nkv) * hd
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn((n, width + 8), generator=g, device="cuda").to(dtype)
    qkv = wide[:, :width]  # rows further apart than their length
    qn = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16() if norm else None
    kn = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16() if norm else None
    rope = rope_table(max(max(kv_lens), 1), rot, theta=500.0)
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    q = paged_append(cache, 0, batch, qkv, rope=rope, rope_pairs=pairs, q_norm=qn, k_norm=kn, eps=1e-5)
    batch.check()
    seq = torch.tensor([b for b, a in enumerate(q_lens) for _ in range(a)], device="cuda")
    pos = torch.tensor([p for a, t in zip(q_lens, kv_lens) for p in range(t - a, t)], device="cuda")
    ok = pos >= 0
    (rq, mq), (rk, mk), rv = append_ref(qkv.contiguous(), nh, nkv, hd, pos.clamp(min=0), rope, pairs, qn, kn, 1e-5)
    check_rounded(q[ok], rq[ok], mq[ok])
    idx = table.long()[seq[ok], pos[ok] // page]
    check_rounded(cache.k[0][idx, :, pos[ok] % page], rk[ok], mk[ok])
    assert torch.equal(cache.v[0][idx, :, pos[ok] % page], rv[ok])
    for pool, old in zip((cache.k, cache.v), before):  # nothing else is touched
        pool[0][idx, :, pos[ok] % page] = 0
        old[0][idx, :, pos[ok] % page] = 0
        assert torch.equal(pool.view(torch.int16), old.view(torch.int16))


def test_rope_table_scaling():
    t = rope_table(64, 32, theta=100.0, device="cpu").double()
    inv = 100.0 ** (-np.arange(0, 32, 2) / 32)
    ang = np.arange(64)[:, None] * inv
    assert np.allclose(t[..., 0], np.cos(ang), atol=1e-7) and np.allclose(t[..., 1], np.sin(ang), atol=1e-7)
    lin = rope_table(64, 32, theta=100.0, scaling={"type": "linear", "factor": 4}, device="cpu")
    assert torch.allclose(lin[::4].double(), t[:16], atol=1e-6)
    ntk = rope_table(64, 32, theta=100.0, scaling={"type": "ntk", "factor": 4}, device="cpu").double()
    assert torch.allclose(ntk[:, 0], t[:, 0])  # the fastest pair stays
    assert np.allclose(ntk[:, -1, 0], np.cos(np.arange(64) * inv[-1] / 4), atol=1e-6)  # the slowest: 4 times slower
    y = rope_table(64, 32, theta=100.0, scaling={"type": "yarn", "factor": 4, "original": 32}, device="cpu").double()
    gain = 0.1 * math.log(4) + 1
    assert torch.allclose((y ** 2).sum(-1).sqrt(), torch.full((64, 16), gain, dtype=torch.float64), atol=1e-6)
    assert np.allclose(y[:, -1, 0], gain * np.cos(np.arange(64) * inv[-1] / 4), atol=1e-6)
    with pytest.raises(ValueError):
        rope_table(8, 7)
    with pytest.raises(ValueError):
        rope_table(8, 8, scaling={"type": "other", "factor": 2})


# ------------------------------------------------ steps, streams and errors --
def test_captured_step_advances_with_the_lengths():
    """update + append + attention captured once and replayed while kv_lens grows on the device."""
    nh, nkv, hd, page = 16, 4, 128, 16
    kv = [30, 3, 200]
    room = [t + 8 for t in kv]
    cache, table, _ = make(nkv, hd, page, [1] * 3, room, seed=11)
    rope = rope_table(300, hd)
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    batch = PagedBatch(cache, [1] * 3, lens, table, num_heads=nh)
    qkv = torch.zeros((3, (nh + 2 * nkv) * hd), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((3, nh, hd), dtype=torch.bfloat16, device="cuda")
    qbuf = torch.zeros_like(out)

    def step():
        batch.update()
        paged_append(cache, 0, batch, qkv, rope=rope, out=qbuf)
        paged_attention(cache, 0, batch, qbuf, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        lens += 1
        qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        now = lens.tolist()
        dense = []
        for b, t in enumerate(now):
            pos = torch.arange(t, device="cuda")
            idx = table[b].long()[pos // page]
            dense.append((cache.k[0][idx, :, pos % page], cache.v[0][idx, :, pos % page]))
            assert torch.equal(dense[-1][1][-1], qkv[b, (nh + nkv) * hd:].view(nkv, hd))
        ref, mag = attention_ref(qbuf, dense, [1] * 3, now, nkv, hd ** -0.5)
        check_attention(out, ref, mag)
    batch.check()


def test_another_stream():
    nh, nkv, hd, page = 16, 16, 128, 16
    cache, table, dense = make(nkv, hd, page, [1, 40], [500, 90], seed=12)
    q = torch.randn((41, nh, hd), device="cuda").bfloat16()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    batch = PagedBatch(cache, [1, 40], [500, 90], table, num_heads=nh, stream=None)
    s.wait_stream(torch.cuda.current_stream())
    out = paged_attention(cache, 0, batch, q, stream=s)
    with torch.cuda.stream(s):
        out2 = paged_attention(cache, 0, batch, q)
    s.synchronize()
    ref, mag = attention_ref(q, dense, [1, 40], [500, 90], nkv, hd ** -0.5)
    check_attention(out, ref, mag)
    assert torch.equal(out, out2)


def test_device_side_errors_are_reported_and_harmless():
    nh, nkv, hd, page = 8, 8, 128, 16
    cache, table, dense = make(nkv, hd, page, [1, 1], [40, 20], seed=13, junk=10 ** 6)
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    # a page id outside the pool: its positions count as zeros, the others as they are
    bad = table.clone()
    bad[1, 1] = 10 ** 6
    batch = PagedBatch(cache, [1, 1], [40, 20], bad, num_heads=nh)
    out = paged_attention(cache, 0, batch, q)
    with pytest.raises(M1MoECudaError, match="0x2"):
        batch.check()
    batch.check()  # reported once
    ref, mag = attention_ref(q[:1], dense[:1], [1], [40], nkv, hd ** -0.5)
    check_attention(out[:1], ref, mag)
    # lengths beyond the page table: an empty batch
    batch = PagedBatch(cache, [1, 1], [40, 10 ** 6], table, num_heads=nh)
    paged_attention(cache, 0, batch, q)
    with pytest.raises(M1MoECudaError, match="0x1"):
        batch.check()
    # a position past the rotation table
    qkv = torch.randn((2, 3 * nh * hd), device="cuda")
    batch = PagedBatch(cache, [1, 1], [40, 20], table, num_heads=nh)
    paged_append(cache, 0, batch, qkv, rope=rope_table(39, hd))
    with pytest.raises(M1MoECudaError, match="0x4"):
        batch.check()


def test_refusals():
    nkv, hd, page = 4, 128, 16
    cache, table, _ = make(nkv, hd, page, [1, 2], [40, 20], seed=14)
    ok = dict(num_heads=8)
    batch = PagedBatch(cache, [1, 2], [40, 20], table, **ok)
    q = torch.zeros((3, 8, hd), dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros((3, 16 * hd), device="cuda")
    rope = rope_table(64, hd)
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, 2], [40, 20], table, num_heads=6)  # not a multiple
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, 2], [40, 20], table, num_heads=17 * nkv)  # more than 16 heads share
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, 2], [40, 20], table, num_heads=8, window=-1)
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, 2], [40, 20], table, num_heads=8, shared_prefix=8)  # not whole pages
    with pytest.raises(ValueError):
        PagedBatch(cache, [1], [40, 20], table, **ok)
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, -2], [40, 20], table, **ok)
    with pytest.raises(ValueError):
        PagedBatch(cache, [1, 2], [40, 20], table.long(), **ok)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(cache.k.float(), cache.v.float())
    with pytest.raises(ValueError):  # page size 24
        k = torch.zeros((1, 4, nkv, 24, hd), dtype=torch.bfloat16, device="cuda")
        PagedBatch(PagedKVCache.from_tensors(k, k.clone()), [1, 2], [4, 4], table[:, :2].contiguous(), **ok)
    with pytest.raises(ValueError):  # head dim 96
        k = torch.zeros((1, 4, nkv, 16, 96), dtype=torch.bfloat16, device="cuda")
        PagedBatch(PagedKVCache.from_tensors(k, k.clone()), [1, 2], [4, 4], table[:, :2].contiguous(), **ok)
    with pytest.raises(ValueError):
        paged_attention(cache, 1, batch, q)  # one layer
    with pytest.raises(TypeError):
        paged_attention(cache, 0, batch, q.float())
    with pytest.raises(ValueError):
        paged_attention(cache, 0, batch, q[:2])
    with pytest.raises(ValueError):
        paged_attention(cache, 0, batch, q.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(M1MoECudaError):
        paged_attention(cache, 0, batch, q, scale=math.nan)
    with pytest.raises(M1MoECudaError):
        paged_attention(cache, 0, batch, q, softcap=-1.0)
    with pytest.raises(TypeError):
        paged_attention(cache, 0, batch, q, out_dtype=torch.float16)
    with pytest.raises(M1MoECudaError):  # 8 bytes off
        flat = torch.zeros(3 * 8 * hd + 8, dtype=torch.bfloat16, device="cuda")
        paged_attention(cache, 0, batch, flat[4:4 + 3 * 8 * hd].view(3, 8, hd))
    with pytest.raises(ValueError):
        paged_append(cache, 0, batch, qkv[:2], rope=rope)
    with pytest.raises(TypeError):
        paged_append(cache, 0, batch, qkv.half(), rope=rope)
    with pytest.raises(ValueError):
        paged_append(cache, 0, batch, qkv, rope=rope.double())
    with pytest.raises(M1MoECudaError):
        paged_append(cache, 0, batch, qkv, rope=rope_table(64, 24))
    with pytest.raises(ValueError):
        paged_append(cache, 0, batch, qkv, rope=rope, q_norm=torch.ones(hd, device="cuda"))


# ----------------------------------------------------------- shared prefix --
@pytest.mark.parametrize("nh,nkv,hd,page,share,q_lens,kv_lens,cap", [
    (16, 16, 128, 16, 16, [1, 1], [17, 40], 0.0),
    (16, 16, 128, 16, 208, [1] * 5, [209, 220, 300, 224, 209], 0.0),
    (32, 8, 128, 64, 1024, [1] * 70, [1025 + 7 * i for i in range(70)], 0.0),
    (32, 8, 64, 32, 4000, [1] * 33, [4001 + i for i in range(33)], 30.0),
    (16, 1, 128, 128, 256, [1] * 40, [257 + 3 * i for i in range(40)], 0.0),
    (24, 8, 64, 16, 640, [1, 3, 2, 1], [641, 643, 900, 700], 0.0),
    (32, 8, 128, 16, 512, [1, 1, 1, 1, 1], [0, 600, 513, 0, 530], 0.0),  # idle slots, the first among them
    (16, 1, 64, 16, 1600, [1], [2000], 0.0),
])
def test_shared_prefix_vs_formula(nh, nkv, hd, page, share, q_lens, kv_lens, cap):
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=21, share=share)
    g = torch.Generator(device="cuda").manual_seed(22)
    q = (1.5 * torch.randn((sum(q_lens), nh, hd), generator=g, device="cuda")).bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, shared_prefix=share)
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, hd ** -0.5, 0, cap)
    for dt in (torch.bfloat16, torch.float32):
        out = paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=dt)
        batch.check()
        check_attention(out, ref, mag)
        assert torch.equal(out, paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=dt))


@pytest.mark.parametrize("why", ["tables differ", "a sequence ends inside it", "windowed", "long new tokens"])
def test_a_prefix_that_cannot_be_shared_changes_nothing(why):
    nh, nkv, hd, page, share = 16, 4, 128, 16, 64
    q_lens, kv_lens, window = [1, 1, 1], [100, 90, 300], 0
    if why == "a sequence ends inside it":
        kv_lens = [100, 64, 300]
    if why == "windowed":
        window = 50
    if why == "long new tokens":
        q_lens = [1, 26, 200]
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=23, share=0 if why == "tables differ" else share)
    q = torch.randn((sum(q_lens), nh, hd), device="cuda").bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, shared_prefix=share, window=window)
    out = paged_attention(cache, 0, batch, q)
    batch.check()
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, hd ** -0.5, window)
    check_attention(out, ref, mag)


# A prefix is read once for the batch where that saves 200 MB of reads; the sizes
# below are above that, in the 16-row form (up to 128 rows a KV head) and the 256-row one.
@pytest.mark.parametrize("nh,nkv,hd,page,share,q_lens,kv_lens,cap", [
    (16, 16, 128, 16, 1024, [1] * 27, [1025 + 5 * i for i in range(27)], 0.0),
    (24, 8, 64, 32, 4064, [1, 2] * 13, [4066 + 9 * i for i in range(26)], 25.0),
    (32, 8, 128, 64, 8192, [1] * 8, [0, 8193, 8400, 0, 8200, 9000, 8193, 8257], 0.0),  # idle slots
    (16, 1, 128, 128, 57344, [1] * 8, [57345 + 40 * i for i in range(8)], 0.0),
    (16, 1, 128, 128, 57344, [1] * 9, [57345 + 40 * i for i in range(9)], 0.0),
])
def test_shared_prefix_read_once(nh, nkv, hd, page, share, q_lens, kv_lens, cap):
    assert (len(q_lens) - 1) * share * nkv * hd * 4 >= 200_000_000
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=24, share=share)
    g = torch.Generator(device="cuda").manual_seed(25)
    q = (1.5 * torch.randn((sum(q_lens), nh, hd), generator=g, device="cuda")).bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, shared_prefix=share)
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, hd ** -0.5, 0, cap)
    for dt in (torch.bfloat16, torch.float32):
        out = paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=dt)
        batch.check()
        check_attention(out, ref, mag)
        assert torch.equal(out, paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=dt))


@pytest.mark.parametrize("why", ["tables differ", "a sequence ends inside it", "no sequence is live"])
def test_a_long_prefix_that_cannot_be_shared_changes_nothing(why):
    nh, nkv, hd, page, share = 32, 8, 128, 64, 8192
    q_lens, kv_lens = [1] * 8, [8193 + 50 * i for i in range(8)]
    if why == "a sequence ends inside it":
        kv_lens[5] = 8192
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=26, share=0 if why == "tables differ" else share)
    q = torch.randn((sum(q_lens), nh, hd), device="cuda").bfloat16()
    lens = [0] * 8 if why == "no sequence is live" else kv_lens
    batch = PagedBatch(cache, q_lens, lens, table, num_heads=nh, shared_prefix=share)
    out = paged_attention(cache, 0, batch, q)
    batch.check()
    if why == "no sequence is live":
        assert not out.any()
        return
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, hd ** -0.5, 0)
    check_attention(out, ref, mag)
