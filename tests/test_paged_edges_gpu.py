"""The paged cache's operators (GPU) where a call meets an edge: values that are not finite, caps far above
the scores, status bits across steps, one token's strides.  Bars as in test_paged_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch
from test_paged_gpu import attention_ref, check_attention, make

from m1moe_b200 import M1MoECudaError, PagedBatch, paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu


def test_a_status_bit_outlives_the_next_plan():
    """A bad page id in one step is still reported after the plan has been made again."""
    nh, nkv, hd, page = 8, 8, 128, 16
    cache, table, _ = make(nkv, hd, page, [1, 1], [40, 20], seed=31)
    good = table.clone()
    table[1, 1] = 10 ** 6
    batch = PagedBatch(cache, [1, 1], [40, 20], table, num_heads=nh)
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    paged_attention(cache, 0, batch, q)
    table.copy_(good)
    for _ in range(3):
        batch.update()
        paged_attention(cache, 0, batch, q)
    with pytest.raises(M1MoECudaError, match="0x2"):
        batch.check()
    batch.update()
    paged_attention(cache, 0, batch, q)
    batch.check()  # reported once


def test_a_new_batch_starts_without_status_bits():
    """Whatever its memory held before: batches made and dropped after raising a bit."""
    nh, nkv, hd, page = 8, 8, 128, 16
    cache, table, _ = make(nkv, hd, page, [1, 1], [40, 20], seed=32)
    bad = torch.full_like(table, 10 ** 6)
    q = torch.randn((2, nh, hd), device="cuda").bfloat16()
    for _ in range(4):
        batch = PagedBatch(cache, [1, 1], [40, 20], bad, num_heads=nh)
        paged_attention(cache, 0, batch, q)
        del batch
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        for kw in ({}, {"stream": s}):
            batch = PagedBatch(cache, [1, 1], [40, 20], table, num_heads=nh, **kw)
            paged_attention(cache, 0, batch, q, **kw)
            batch.check(**kw)
            del batch


@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e8, 3e38])
@pytest.mark.parametrize("hd,q_lens,kv_lens", [(128, [1, 1, 1], [1, 700, 33]), (64, [2, 1], [90, 64]),
                                               (128, [70, 200], [300, 200]), (64, [130], [130])])
def test_caps_far_above_the_scores(hd, q_lens, kv_lens, cap):
    """cap tanh(s / cap) of scores between a ten-thousandth and a few times the cap: as the cap grows the
    result is the uncapped one.  Errors of tanh are relative (6e-7 at most), so scores of up to about 20 are
    off by about 1e-5, far inside the bar's 2^-11."""
    nh, nkv = 16, 4
    cache, table, dense = make(nkv, hd, 16, q_lens, kv_lens, seed=33)
    q = (3 * torch.randn((sum(q_lens), nh, hd), device="cuda")).bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    out = paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=torch.float32)
    batch.check()
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 1 / math.sqrt(hd), 0, cap)
    check_attention(out, ref, mag)


def attention_seen(q, dense, q_lens, kv_lens, nkv, scale, window):
    """The formula in 64 bits, its sums over the positions a row sees and nothing else; and sum w |v|."""
    ref = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag, at, group = torch.zeros_like(ref), 0, q.shape[1] // nkv
    for (k, v), a, t in zip(dense, q_lens, kv_lens):
        for i in range(a):
            hi = t - a + i
            lo = max(0, hi - window + 1) if window else 0
            ks, vs = k[lo:hi + 1].double(), v[lo:hi + 1].double()
            x = q[at + i].double().view(nkv, group, -1)
            w = torch.softmax(torch.einsum("hgd,thd->hgt", x, ks) * scale, -1)
            ref[at + i] = torch.einsum("hgt,thd->hgd", w, vs).reshape(-1, q.shape[2])
            mag[at + i] = torch.einsum("hgt,thd->hgd", w, vs.abs()).reshape(-1, q.shape[2])
        at += a
    return ref, mag


@pytest.mark.parametrize("nh,nkv,hd,page,q_lens,kv_lens,window", [
    (16, 4, 128, 16, [4, 1, 3], [30, 50, 3], 0),            # 16-row items
    (8, 4, 64, 32, [8, 2], [100, 17], 3),
    (16, 4, 128, 16, [60, 1, 200], [60, 300, 290], 0),      # 256-row items, whole tiles and edges
    (16, 4, 128, 64, [300, 40], [700, 40], 50),
    (4, 4, 64, 128, [270], [270], 0),
    (32, 2, 128, 16, [70], [3000], 0),                      # an item cut over many runs
])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(nh, nkv, hd, page, q_lens, kv_lens, window, value):
    """A V element that is no finite number belongs to the sums of the rows that see its position; the
    rows before it (and those whose window has passed it) are what they were."""
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=34)
    q = torch.randn((sum(q_lens), nh, hd), device="cuda").bfloat16()
    dense = [(k.clone(), v.clone()) for k, v in dense]
    for b, (a, t) in enumerate(zip(q_lens, kv_lens)):
        # in the middle of the new tokens, at the last one, and (windowed: passed by some rows) before them
        for pos, col in ((t - a + a // 2, 3), (t - 1, hd - 1), (max(0, t - a - 1), hd // 2)):
            if pos == 0:
                continue
            dense[b][1][pos, nkv - 1, col] = value
            cache.v[0][table[b, pos // page].long(), nkv - 1, pos % page, col] = value
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=window)
    ref, mag = attention_seen(q, dense, q_lens, kv_lens, nkv, 1 / math.sqrt(hd), window)
    finite = ref.isfinite()
    assert finite.any() and not finite.all()
    for dt in (torch.float32, torch.bfloat16):
        out = paged_attention(cache, 0, batch, q, out_dtype=dt)
        batch.check()
        assert torch.equal(out.isfinite(), finite)
        assert torch.equal(out[~finite].nan_to_num(7.0, 8.0, 9.0).double(), ref[~finite].nan_to_num(7.0, 8.0, 9.0))
        check_attention(torch.where(finite, out, 0), torch.where(finite, ref, 0), torch.where(finite, mag, 0))


def test_one_token_may_have_any_row_stride():
    """A dimension of one row has no stride: what the tensor says of it is not looked at."""
    nh, nkv, hd, page = 4, 2, 128, 16
    cache, table, _ = make(nkv, hd, page, [1], [20], seed=35)
    rope = rope_table(32, hd)
    batch = PagedBatch(cache, [1], [20], table, num_heads=nh)
    qkv = torch.randn((1, (nh + 2 * nkv) * hd), device="cuda").bfloat16()
    ref = paged_append(cache, 0, batch, qkv, rope=rope)
    odd = qkv.view(-1, 1).t()
    assert odd.stride() == (1, 1)
    assert torch.equal(paged_append(cache, 0, batch, odd, rope=rope), ref)
    # one head: the stride between heads is not looked at either
    cache, table, dense = make(1, hd, page, [2], [20], seed=36)
    batch = PagedBatch(cache, [2], [20], table, num_heads=1)
    q = torch.randn((1, 2, hd), device="cuda").bfloat16().transpose(0, 1)
    assert q.stride() == (hd, 2 * hd, 1)
    out = paged_attention(cache, 0, batch, q)
    assert torch.equal(out, paged_attention(cache, 0, batch, q.contiguous()))


@pytest.mark.parametrize("nh,nkv,hd,page,q_lens,kv_lens,window,cap", [
    (16, 4, 128, 16, [4, 1, 3], [30, 50, 3], 0, 0.0), (8, 4, 64, 32, [8, 2], [100, 17], 3, 20.0),
    (16, 4, 128, 16, [60, 1, 200], [60, 300, 290], 0, 30.0), (16, 4, 128, 64, [300, 40], [700, 40], 50, 0.0)])
def test_keys_that_are_not_finite_reach_only_the_rows_that_see_them(nh, nkv, hd, page, q_lens, kv_lens, window, cap):
    """A NaN key makes the rows that see it NaN, throughout their head, and no others."""
    cache, table, dense = make(nkv, hd, page, q_lens, kv_lens, seed=37)
    q = torch.randn((sum(q_lens), nh, hd), device="cuda").bfloat16()
    ref, mag = attention_ref(q, dense, q_lens, kv_lens, nkv, 1 / math.sqrt(hd), window, cap)
    sees = torch.zeros((sum(q_lens), nh), dtype=torch.bool, device="cuda")
    at, group = 0, nh // nkv
    for b, (a, t) in enumerate(zip(q_lens, kv_lens)):
        bad = t - a + a // 2
        cache.k[0][table[b, bad // page].long(), 0, bad % page, 5] = math.nan
        pos = torch.arange(t - a, t, device="cuda")
        see = pos >= bad
        if window:
            see &= pos - bad < window
        sees[at:at + a, :group] = see[:, None]
        at += a
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=window)
    for dt in (torch.float32, torch.bfloat16):
        out = paged_attention(cache, 0, batch, q, softcap=cap, out_dtype=dt)
        batch.check()
        assert torch.equal(out.isnan(), sees[..., None].expand_as(out))
        keep = ~sees[..., None].expand_as(out)
        check_attention(torch.where(keep, out, 0), torch.where(keep, ref, 0), torch.where(keep, mag, 0))


@pytest.mark.parametrize("nh,nkv,hd,q_lens,kv_lens,window", [
    (16, 4, 128, [4], [30], 0), (8, 4, 64, [8], [100], 1), (8, 2, 128, [60], [300], 0), (4, 4, 64, [270], [270], 2)])
def test_a_hidden_nan_does_not_change_an_infinite_result(nh, nkv, hd, q_lens, kv_lens, window):
    """Rows whose own value is infinite beside later ones that are NaN or of the other sign, in one column."""
    cache, table, dense = make(nkv, hd, 16, q_lens, kv_lens, seed=38)
    t, a = kv_lens[0], q_lens[0]
    v = dense[0][1].clone()
    at = t - a + a // 2
    for pos, value in ((at, math.inf), (at + 1, -math.inf if window == 1 else math.inf), (t - 1, math.nan)):
        v[pos, 1, 7] = value
        cache.v[0][table[0, pos // 16].long(), 1, pos % 16, 7] = value
    q = torch.randn((a, nh, hd), device="cuda").bfloat16()
    ref, mag = attention_seen(q, [(dense[0][0], v)], q_lens, kv_lens, nkv, 1 / math.sqrt(hd), window)
    finite = ref.isfinite()
    assert ref.isinf().any() and ref.isnan().any()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=window)
    out = paged_attention(cache, 0, batch, q, out_dtype=torch.float32)
    batch.check()
    assert torch.equal(out[~finite].nan_to_num(7.0, 8.0, 9.0).double(), ref[~finite].nan_to_num(7.0, 8.0, 9.0))
    check_attention(torch.where(finite, out, 0), torch.where(finite, ref, 0), torch.where(finite, mag, 0))


@pytest.mark.parametrize("nh,nkv,hd,q_lens,kv_lens", [(16, 4, 128, [4, 3], [2, 1]), (8, 4, 64, [331, 20], [134, 20]),
                                                      (4, 4, 128, [600], [40])])
def test_rows_before_position_0_stay_zero(nh, nkv, hd, q_lens, kv_lens):
    """Tokens that a sequence is too short for see nothing, whatever the positions beside them hold."""
    cache, table, _ = make(nkv, hd, 16, q_lens, kv_lens, seed=39)
    for b, t in enumerate(kv_lens):
        cache.v[0][table[b, (t - 1) // 16].long(), :, (t - 1) % 16] = math.nan
    q = torch.randn((sum(q_lens), nh, hd), device="cuda").bfloat16()
    batch = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh)
    out = paged_attention(cache, 0, batch, q)
    batch.check()
    at = 0
    for a, t in zip(q_lens, kv_lens):
        rows = out[at:at + a]
        assert not rows[:max(0, a - t)].any() and rows[:a - 1].isfinite().all() and rows[a - 1].isnan().all()
        at += a
