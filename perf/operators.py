"""Serving operators over a paged key/value cache, and the sampler: what is measured.

Four operators, in their plain form (elementary torch operations in 32 bits) and, with
`own` set, as calls of this package:

  append   per-head RMSNorm of queries and keys, rotary position embedding and the store of
           the new keys and values into the pages of a ragged batch's sequences
  attend   causal attention of a ragged batch's new tokens over their paged sequences
           (one token per sequence up to whole prompts; optional sliding window and tanh cap)
  shared   the same for one token per sequence when the batch shares a long prefix (a system
           prompt) whose pages are the same for every sequence
  sample   temperature, top-k, top-p and min-p sampling of a batch of logit rows with one
           given uniform number per row

The cache of one layer is two bf16 arrays [pages][kv heads][page size][head dim]; a sequence
is a row of a page table; its last tokens are the batch's new ones.
"""
import math
import random

import torch

own = False

# (query heads, key/value heads): the framework's two model shapes, then group sizes of 2, 3 and 16
HEADS = ((16, 16), (32, 8), (8, 4), (24, 8), (16, 1))


# ------------------------------------------------------------------ the cases --


def listed():
    return [
        # One new token of a chat at the 2048-token context of the OLMoE-shaped decode step: latency.
        _batch("append", "append-token", 16, 16, page=16, q=(1, 1), ctx=(2047, 2047), dtype="f32", norm=True),
        # A continuous-batching decode step of 64 Mixtral-shaped sequences.
        _batch("append", "append-decode-64", 32, 8, n=64, page=64, q=(1, 1), ctx=(37, 16000), dtype="bf16", seed=1),
        # Nine ragged prompts admitted together; adjacent pairs rotated, half of each head only.
        _batch("append", "append-prompts", 32, 8, n=9, page=32, q=(61, 4099), ctx=(0, 900), dtype="bf16", norm=True,
               rot=64, pairs=True, seed=2),
        # The attention of the single chat's token above.
        _batch("attend", "attend-token", 16, 16, page=16, q=(1, 1), ctx=(2047, 2047)),
        # The attention of a 64-sequence decode step, lengths from tens to 16 thousand.
        _batch("attend", "attend-decode-64", 32, 8, n=64, page=64, q=(1, 1), ctx=(37, 16000), seed=1),
        # Decode steps and prompt chunks in one batch, with a sliding window and capped scores.
        _batch("attend", "attend-mixed", 16, 16, n=12, page=32, q=(1, 1023), ctx=(0, 5000), window=2048, cap=50.0,
               seed=3),
        # One long prompt of a Mixtral-shaped model.
        _batch("attend", "attend-prompt-8k", 32, 8, page=64, q=(8192, 8192), ctx=(0, 0)),
        # Sixteen chats behind one 1500-token system prompt.
        _batch("shared", "shared-16", 16, 16, n=16, page=16, prefix=1504, q=(1, 1), ctx=(5, 300), seed=4),
        # Two hundred requests about one long document.
        _batch("shared", "shared-200", 32, 8, n=200, page=64, prefix=16384, q=(1, 1), ctx=(20, 1500), seed=5),
        # The next token of one chat, OLMoE-sized vocabulary.
        {"op": "sample", "name": "sample-one", "rows": 1, "vocab": 50304, "dtype": "f32", "seed": 0},
        # A step of a batch of 192 requests, each with its own settings, Mixtral-sized vocabulary.
        {"op": "sample", "name": "sample-192", "rows": 192, "vocab": 32000, "dtype": "f32", "seed": 1},
        # Many candidates for each of a few prompts over a large odd vocabulary, bf16 logits.
        {"op": "sample", "name": "sample-vocab-150k", "rows": 48, "vocab": 150001, "dtype": "bf16", "seed": 2},
    ]


def draw(rng):
    """One more case of the same ranges, no dearer than the largest listed one of its operator."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        c = _draw_any(rng)
        if _cost(c) <= most[c["op"]]:
            return c


def _draw_any(rng):
    op = rng.choice(("append", "append", "attend", "attend", "attend", "shared", "shared", "sample", "sample"))
    seed = rng.randrange(1 << 20)
    if op == "sample":
        return {"op": op, "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 1000, 200000),
                "dtype": rng.choice(("f32", "bf16")), "seed": seed}
    nh, nkv = rng.choice(HEADS)
    hd = rng.choice((128, 128, 64))
    page = rng.choice((16, 32, 64, 128))
    if op == "shared":
        prefix = page * max(1, _log_int(rng, 256, 16384) // page)
        return _batch(op, None, nh, nkv, hd=hd, n=_log_int(rng, 2, 256), page=page, prefix=prefix, q=(1, 1),
                      ctx=(0, _log_int(rng, 16, 2000)), cap=rng.choice((0.0, 0.0, 30.0)), seed=seed)
    n = _log_int(rng, 1, 128)
    q = (1, 1) if rng.random() < 0.5 else (1, _log_int(rng, 2, 4100))
    ctx = (0, _log_int(rng, 1, 20000))
    if op == "append":
        return _batch(op, None, nh, nkv, hd=hd, n=n, page=page, q=q, ctx=ctx, dtype=rng.choice(("f32", "bf16")),
                      norm=rng.random() < 0.5, rot=rng.choice((hd, hd, hd // 2)), pairs=rng.random() < 0.5, seed=seed)
    return _batch(op, None, nh, nkv, hd=hd, n=n, page=page, q=q, ctx=ctx,
                  window=rng.choice((0, 0, _log_int(rng, 1, 4096))), cap=rng.choice((0.0, 0.0, 30.0)), seed=seed)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _batch(op, name, nh, nkv, hd=128, n=1, page=16, prefix=0, q=(1, 1), ctx=(0, 0), dtype="bf16", norm=False, rot=0,
           pairs=False, window=0, cap=0.0, seed=0):
    c = {"op": op, "heads": nh, "kv_heads": nkv, "head_dim": hd, "seqs": n, "page": page, "q_min": q[0], "q_max": q[1],
         "ctx_min": ctx[0], "ctx_max": ctx[1], "seed": seed}
    if name:
        c["name"] = name
    if op == "append":
        c.update(dtype=dtype, norm=norm, rot=rot or hd, pairs=pairs)
    else:
        c.update(window=window, cap=cap)
    if op == "shared":
        c["prefix"] = prefix
    return c


def _lengths(c):
    """(new tokens, all tokens) of each sequence: the first has the most of both, the others are
    spread over the logarithm of their ranges."""
    rng = random.Random(c["seed"])
    q, kv = [c["q_max"]], [c["ctx_max"]]
    for _ in range(c["seqs"] - 1):
        q.append(_log_int(rng, c["q_min"], c["q_max"]))
        kv.append(_log_int(rng, c["ctx_min"] + 1, c["ctx_max"] + 1) - 1)
    return q, [c.get("prefix", 0) + a + b for a, b in zip(q, kv)]


def work(c):
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        # a maximum, a scaled exponential and a sum for each logit
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + c["rows"] * 24, "flops": 4 * n}
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    q, kv = _lengths(c)
    tokens = sum(q)
    table = 4 * sum(-(-t // c["page"]) for t in kv)
    if c["op"] == "append":
        size = 4 if c["dtype"] == "f32" else 2
        width = (nh + 2 * nkv) * hd
        # the projections in; the queries and the cache rows out; one row of the rotation table a token
        return {"bytes": tokens * (width * size + width * 2 + c["rot"] * 4) + table,
                "flops": tokens * (nh + nkv) * (3 * c["rot"] + (4 * hd if c["norm"] else 0))}
    window = c["window"]
    pairs = rows = 0
    for a, t in zip(q, kv):
        first = t - a
        if window:
            pairs += sum(min(p + 1, window) for p in range(first, t))
            rows += t - max(0, first + 1 - window)
        else:
            pairs += (first + 1 + t) * a // 2
            rows += t
    rows -= c.get("prefix", 0) * (c["seqs"] - 1)  # the shared rows are read once
    return {"bytes": rows * nkv * hd * 4 + tokens * nh * hd * 4 + table, "flops": 4 * pairs * nh * hd}


def _cost(c):
    w = work(c)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


# ----------------------------------------------------------------- the inputs --


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + c["seed"])
    if c["op"] == "sample":
        return _prepare_sample(c, g)
    nh, nkv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    q_lens, kv_lens = _lengths(c)
    prefix = c.get("prefix", 0)
    # pages in a random order, as a long-running server's free list gives them; the prefix's are shared
    need = [-(-t // page) for t in kv_lens]
    shared = prefix // page
    total = shared + sum(x - shared for x in need)
    pages = total + 3  # some belong to nobody
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, x in enumerate(need):
        table[b, :shared] = order[:shared]
        table[b, shared:x] = order[at:at + x - shared]
        at += x - shared
    shape = (pages, nkv, page, hd)
    k, v = _normal(g, shape), _normal(g, shape)
    tokens = sum(q_lens)
    s = {"case": c, "table": table, "k": k, "v": v, "q_lens": q_lens, "kv_lens": kv_lens}
    if c["op"] == "append":
        width = (nh + 2 * nkv) * hd
        x = torch.randn((tokens, width), generator=g, device="cuda")
        s["qkv"] = x if c["dtype"] == "f32" else x.bfloat16()
        s["q_norm"] = s["k_norm"] = None
        if c["norm"]:
            s["q_norm"] = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).bfloat16()
            s["k_norm"] = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).bfloat16()
        # the model's cosines and sines, position by position: made once when the model is loaded
        angle = torch.arange(max(kv_lens), device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"]))
        s["rope"] = torch.stack((angle.cos(), angle.sin()), dim=-1).float()
    else:
        # queries a few times the keys' scale: some heads attend to little, some to much
        q = torch.randn((tokens, nh, hd), generator=g, device="cuda")
        s["q"] = (q * (0.5 + 2.5 * torch.rand((1, nh, 1), generator=g, device="cuda"))).bfloat16()
    if own:
        from m1moe_b200.paged import PagedBatch, PagedKVCache

        cache = PagedKVCache.from_tensors(k[None], v[None])
        s["cache"] = cache
        s["batch"] = PagedBatch(cache, q_lens, kv_lens, table, num_heads=nh, window=c.get("window", 0),
                                shared_prefix=prefix)
    return s


def _normal(g, shape):
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    flat = x.view(-1)
    for a in range(0, flat.numel(), 1 << 28):
        b = min(flat.numel(), a + (1 << 28))
        flat[a:b].normal_(generator=g)
    return x


def _prepare_sample(c, g):
    rows, vocab = c["rows"], c["vocab"]
    # a language model's logits: a broad bulk and, in each row, some candidates far above it
    x = 2.2 * torch.randn((rows, vocab), generator=g, device="cuda")
    n = min(40, vocab)
    best = torch.randint(0, vocab, (rows, n), generator=g, device="cuda")
    x.scatter_(1, best, 6 + 2.5 * torch.randn((rows, n), generator=g, device="cuda"))
    x[:, vocab // 2:vocab // 2 + 3] = -math.inf  # forbidden tokens
    pick = torch.rand((4, rows), generator=g, device="cuda")
    one = {"dtype": torch.float32, "device": "cuda"}
    s = {"case": c, "logits": x if c["dtype"] == "f32" else x.bfloat16(),
         "u": torch.rand(rows, generator=g, device="cuda")}
    # each request has its own settings; about a sixth are greedy, some leave a filter off
    temp = torch.tensor([0.0, 0.6, 0.7, 0.8, 1.0, 1.3], **one)
    s["temperature"] = temp[(pick[0] * 6).long()] if rows > 1 else torch.tensor([0.7], **one)
    ks = torch.tensor([0, 20, 40, 50, 1000], dtype=torch.int32, device="cuda")
    s["top_k"] = ks[(pick[1] * 5).long()]
    ps = torch.tensor([1.0, 0.8, 0.9, 0.95, 0.999], **one)
    s["top_p"] = ps[(pick[2] * 5).long()]
    ms = torch.tensor([0.0, 0.0, 0.02, 0.1], **one)
    s["min_p"] = ms[(pick[3] * 4).long()]
    return s


# ------------------------------------------------------------------ the calls --


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    if c["op"] == "append":
        return _plain_append(s, c)
    if c["op"] == "sample":
        return _plain_sample(s)
    return _plain_attend(s, c)


def _own(s, c):
    if c["op"] == "append":
        from m1moe_b200.paged import paged_append

        q = paged_append(s["cache"], 0, s["batch"], s["qkv"], rope=s["rope"], rope_pairs=c["pairs"],
                         q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-5)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "sample":
        from m1moe_b200.sampling import sample

        return sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"])
    from m1moe_b200.paged import paged_attention

    return paged_attention(s["cache"], 0, s["batch"], s["q"], softcap=c["cap"])


def _rows_of(s, b, t):
    """Pool rows of positions 0..t-1 of sequence b: (page, offset in it)."""
    page = s["case"]["page"]
    at = torch.arange(t, device="cuda")
    return s["table"][b].long()[at // page], at % page


def _rms(x, w, eps):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(x.dtype)


def _rotate(x, cs, pairs):
    """x [tokens][heads][dim]; cs [tokens][rot/2][2]: the first rot elements of each head."""
    half = cs.shape[1]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    if pairs:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), dim=-1).flatten(-2) if pairs else torch.cat((ra, rb), dim=-1)
    return torch.cat((r, x[..., 2 * half:]), dim=-1)


def _plain_append(s, c):
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    where, pos = [], []
    for b, (a, t) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        p = torch.arange(t - a, t, device="cuda")
        pos.append(p)
        where.append(s["table"][b].long()[p // c["page"]])
    pos, where = torch.cat(pos), torch.cat(where)
    cs = s["rope"][pos]
    q = _rotate(_rms(x[:, :nh], s["q_norm"], 1e-5), cs, c["pairs"])
    k = _rotate(_rms(x[:, nh:nh + nkv], s["k_norm"], 1e-5), cs, c["pairs"])
    s["k"][where, :, pos % c["page"]] = k.bfloat16()
    s["v"][where, :, pos % c["page"]] = x[:, nh + nkv:].bfloat16()
    return {"q": q.bfloat16(), "k": s["k"], "v": s["v"]}


def _plain_attend(s, c):
    nh, nkv, hd, window, cap = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["cap"]
    out = torch.empty_like(s["q"])
    scale, at = 1.0 / math.sqrt(hd), 0
    for b, (a, t) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        where, off = _rows_of(s, b, t)
        k = s["k"][where, :, off].float().permute(1, 0, 2)  # [kv heads][t][dim]
        v = s["v"][where, :, off].float().permute(1, 0, 2)
        for i in range(0, a, 512):  # blocks of queries, to bound the scores' memory
            n = min(512, a - i)
            first = t - a + i
            lo = max(0, first + 1 - window) if window else 0
            hi = first + n
            q = s["q"][at + i:at + i + n].float().view(n, nkv, nh // nkv, hd).permute(1, 2, 0, 3).reshape(nkv, -1, hd)
            x = torch.matmul(q, k[:, lo:hi].transpose(1, 2)) * scale
            if cap:
                x = cap * torch.tanh(x / cap)
            if n > 1:
                qp = torch.arange(first, hi, device="cuda")[:, None]
                kp = torch.arange(lo, hi, device="cuda")[None]
                hide = kp > qp
                if window:
                    hide = hide | (kp <= qp - window)
                x = x.view(nkv, nh // nkv, n, hi - lo).masked_fill(hide, -math.inf).view(nkv, -1, hi - lo)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(x, v[:, lo:hi]) / x.sum(-1, keepdim=True)
            out[at + i:at + i + n] = o.view(nkv, nh // nkv, n, hd).permute(2, 0, 1, 3).reshape(n, nh, hd).bfloat16()
        at += a
    return out


def _mul24(total, f):
    """floor(total * f / 2^24) of whole numbers: total < 2^62, 0 <= f <= 2^24."""
    return (total >> 24) * f + (((total & 0xFFFFFF) * f) >> 24)


def _plain_sample(s):
    """A token's weight is the whole part of 2^36 exp((logit - largest) / temperature), so that every
    sum below is a sum of whole numbers and does not depend on its order.  Tokens are ranked by logit
    (ties: the lower index first).  Kept are the top_k first ones (0: all); of these the shortest run
    of first ones whose weight reaches the part top_p of theirs; of these the ones with
    exp(...) >= min_p.  The token is the first, by index, whose running kept weight exceeds the part
    u of the kept weight.  Temperature 0 takes the first rank, a row of -inf gives -1."""
    x = s["logits"].float()
    rows, vocab = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    temp = s["temperature"][:, None]
    e = torch.where(x == top, 1.0, torch.exp((x - top) * (1.0 / temp)))
    w = (e * float(1 << 36)).long()
    rank = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, rank)
    place = torch.arange(vocab, device="cuda")[None]
    k = s["top_k"][:, None].long()
    keep = (place < k) | (k <= 0)
    keep = keep & ((temp > 0) | (place == 0))
    ws = torch.where(keep, ws, 0)
    part = (s["top_p"][:, None] * float(1 << 24)).long().clamp(0, 1 << 24)
    need = _mul24(ws.sum(-1, keepdim=True), part)
    before = ws.cumsum(-1) - ws
    keep = keep & ((before < need) | (place == 0) | (part == 1 << 24))
    keep = keep & (e.gather(1, rank) >= s["min_p"][:, None])
    w = torch.zeros_like(w).scatter_(1, rank, torch.where(keep, ws, 0))
    run = w.cumsum(-1)
    u = (s["u"][:, None] * float(1 << 24)).long().clamp(0, (1 << 24) - 1)
    token = (run <= _mul24(run[:, -1:], u)).sum(-1)
    return torch.where(top[:, 0] == -math.inf, -1, token).int()


# ------------------------------------------------------------ from definition --


def exact(c, seed):
    """What `run` returns, in 64 bits from the definitions."""
    s = prepare(c, seed)
    if c["op"] == "append":
        return _exact_append(s, c)
    if c["op"] == "sample":
        return _exact_sample(s)
    return _exact_attend(s, c)


def _exact_append(s, c):
    nh, nkv, hd, page, rot = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["rot"]
    x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
    pos = torch.tensor([p for a, t in zip(s["q_lens"], s["kv_lens"]) for p in range(t - a, t)], device="cuda")
    seq = torch.tensor([b for b, a in enumerate(s["q_lens"]) for _ in range(a)], device="cuda")
    first = torch.arange(0, rot, 2, device="cuda") if c["pairs"] else torch.arange(rot // 2, device="cuda")
    second = first + (1 if c["pairs"] else rot // 2)
    # the rotation as complex multiplication by the table's entries
    z = torch.view_as_complex(s["rope"].double().contiguous())[pos][:, None]

    def turned(h, w):
        if w is not None:
            h = h * w.double() / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / hd + 1e-5)
        r = torch.complex(h[..., first], h[..., second]) * z
        h = h.clone()
        h[..., first], h[..., second] = r.real, r.imag
        return h

    k, v = s["k"].double(), s["v"].double()
    slot = s["table"].long()[seq, pos // page]
    k[slot, :, pos % page] = turned(x[:, nh:nh + nkv], s["k_norm"])
    v[slot, :, pos % page] = x[:, nh + nkv:]
    return {"q": turned(x[:, :nh], s["q_norm"]), "k": k, "v": v}


def _exact_attend(s, c):
    if work(c)["flops"] > 1.5e12:
        return None
    nh, nkv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (a, t) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        table = s["table"][b, :-(-t // page)].long()
        key_at = torch.arange(t, device="cuda")
        for h in range(nkv):
            k = s["k"][table, h].reshape(-1, hd)[:t].double()
            v = s["v"][table, h].reshape(-1, hd)[:t].double()
            group = range(h * nh // nkv, (h + 1) * nh // nkv)
            step = max(1, (1 << 27) // (t * len(group)))
            for i in range(0, a, step):
                n = min(step, a - i)
                q_at = torch.arange(t - a + i, t - a + i + n, device="cuda")[:, None, None]
                sees = key_at <= q_at
                if c["window"]:
                    sees = sees & (q_at - key_at < c["window"])
                q = s["q"][at + i:at + i + n, group.start:group.stop].double()
                x = torch.einsum("qgd,kd->qgk", q, k) / math.sqrt(hd)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                p = torch.softmax(torch.where(sees, x, -math.inf), dim=-1)
                out[at + i:at + i + n, group.start:group.stop] = torch.einsum("qgk,kd->qgd", p, v)
        at += a
    return out


def _exact_sample(s):
    """Probabilities in 64 bits, rows one by one; None where a row lies so near a boundary of the
    filters or of the token's interval that rounding in 32 bits may rightly decide it otherwise."""
    answers = [_sample_rows(s, shift) for shift in (0.0, -3e-6, 3e-6)]
    return torch.tensor(answers[0], dtype=torch.int32) if answers[0] == answers[1] == answers[2] else None


def _sample_rows(s, shift):
    out = []
    x = s["logits"].double().cpu()
    rows = zip(x, *(s[k].double().cpu().tolist() for k in ("temperature", "top_k", "top_p", "min_p", "u")))
    for row, temp, k, p, least, u in rows:
        order = torch.sort(row, descending=True, stable=True).indices
        if row[order[0]] == -math.inf:
            out.append(-1)
            continue
        if temp == 0:
            out.append(int(order[0]))
            continue
        prob = torch.softmax(row[order] / temp, 0)
        n = int(k) if k > 0 else len(prob)
        prob[n:] = 0
        prob = prob / prob.sum()
        if p < 1:
            reached = torch.nonzero(prob.cumsum(0) >= p * (1 + shift))
            prob[int(reached[0]) + 1 if len(reached) else n:] = 0
        prob = torch.where(prob >= least * (1 + shift) * prob[0], prob, 0.0)
        by_index = torch.zeros_like(prob).index_copy_(0, order, prob).cumsum(0)
        out.append(int(torch.searchsorted(by_index, (u + shift) * float(by_index[-1]), right=True)))
    return out
