"""Performance cases of the paged INT4 KV cache: rotate-and-append, read back, attention.

Each case is one pass of a serving step through one operator, over the shapes a
server meets: single tokens, token batches of ragged length, prompts.  ``run``
computes it with elementary torch operations, or, where ``own`` is set, with
``spectra_b200.paged``.

A cache is one byte tensor [pages, kv_heads, page / 16, tile_bytes].  A tile holds
16 tokens of one head, D = 32 G features each (offsets in bytes):
  key codes    16*D/2  [2 blocks of 8 tokens][8 tokens][4 words c][G]: word c of group g holds
                       features 8c..8c+7 of the group, low nibble first
  value codes  16*D/2  [2 blocks][8 lanes l][4 token pairs][G]: features 4l..4l+3 of group g of the
                       even token in the low half of the word, of the odd token in the high half
  key scales   fp16 [16][G],   value scales  fp16 [8 token pairs][G][2]
  key zeros    u8   [16][G],   value zeros   u8   [8 token pairs][G][2]
and a code q stands for (q - zero) * scale.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, **kw):
    c = dict(name=name, op=op, dtype="bf16", heads=32, kv_heads=8, head_dim=128, page=64, batch=1, ctx=1024, new=1,
             ragged=0, rotary=0, interleaved=False, causal=True, window=0, softcap=0.0, alibi=False)
    c.update(kw)
    return c


def listed():
    return [
        # one token of a 1B model's layer: pure latency
        _case("append-one", "append", head_dim=64, ctx=1281, rotary=64),
        # one decode step of a busy server: 128 sequences of any length, one token each
        _case("append-128-sequences", "append", batch=128, ctx=8192, ragged=1, rotary=128),
        # ragged prompts, fp16, neighbouring pairs rotated in a part of the head, small pages
        _case("append-prompts-fp16", "append", dtype="fp16", heads=16, kv_heads=4, head_dim=96, page=16, batch=7,
              ctx=2049, new=2049, ragged=2, rotary=64, interleaved=True),
        # one long prompt of a 70B-shaped layer
        _case("append-prompt-16384", "append", heads=64, ctx=16384, new=16384, rotary=128),
        # one token after a prompt of 1024, 1B-shaped layer: latency
        _case("attend-one-1024", "attend", head_dim=64, ctx=1024),
        # one token of one long conversation, 8B-shaped layer: the cache has to be split
        _case("attend-one-131072", "attend", ctx=131072),
        # decode step of a busy server on a 70B-shaped layer
        _case("attend-64-sequences", "attend", heads=64, batch=64, ctx=8192, ragged=3),
        # wide heads with a score cap and a sliding window, fp16, odd lengths, small pages
        _case("attend-window-cap-fp16", "attend", dtype="fp16", heads=8, kv_heads=4, head_dim=256, page=16, batch=33,
              ctx=3001, ragged=4, window=1024, softcap=50.0),
        # checking up to five drafted tokens per sequence, distance bias in place of rotation
        _case("attend-verify-bias", "attend", batch=8, ctx=6001, new=5, ragged=5, alibi=True),
        # a prompt of 1024 on an 8B-shaped layer
        _case("attend-prompt-1024", "attend", ctx=1024, new=1024),
        # ragged prompts with a score cap, every query head with heads of 64
        _case("attend-prompts-cap-fp16", "attend", dtype="fp16", heads=64, head_dim=64, batch=6, ctx=2501, new=2501,
              ragged=6, softcap=30.0),
        # a chunk of a long prompt: 4096 new tokens that look back at 16384
        _case("attend-chunk-4096", "attend", ctx=16384, new=4096),
    ]


_HEADS = [(32, 8, 64), (32, 8, 128), (64, 8, 128), (4, 2, 64), (16, 16, 64), (32, 32, 128), (16, 4, 96), (8, 4, 256),
          (8, 1, 32), (40, 8, 128), (12, 1, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice(_HEADS)
    op = rng.choice(["append", "attend", "attend", "attend"])
    form = rng.choice(["one", "one", "few", "prompt"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), heads=heads, kv_heads=kv_heads, head_dim=dim,
             page=rng.choice([16, 32, 64, 128]), ragged=rng.randrange(1, 1000), rotary=0, interleaved=False,
             causal=True, window=0, softcap=0.0, alibi=False)
    if form == "one":
        batch, ctx, new = _log(rng, 1, 200), _log(rng, 16, 131072), 1
    elif form == "few":
        batch, ctx, new = _log(rng, 1, 64), _log(rng, 32, 32768), rng.randrange(2, 33)
    else:
        batch, new = _log(rng, 1, 12), _log(rng, 64, 4096)
        ctx = new if rng.random() < 0.6 else new + _log(rng, 1, 12288)
    # no more than the largest listed case: cached values, and pairs of a query and a key
    ctx = max(new, min(ctx, 500_000_000 // (batch * kv_heads * dim)))
    while batch > 1 and batch * kv_heads * dim * ctx > 500_000_000:
        batch //= 2
    if op == "attend":
        each = heads * max(dim, 128)
        while batch > 1 and batch * each * new * ctx > 32 * 128 * 4096 * 16384:
            batch //= 2
        while batch * each * new * ctx > 32 * 128 * 4096 * 16384:
            new, ctx = max(1, new // 2), max(1, new // 2, ctx // 2)
    c.update(batch=batch, ctx=ctx, new=new)
    if op == "append":
        c.update(rotary=rng.choice([dim, dim, dim // 2, 0]), interleaved=rng.random() < 0.3)
    else:
        c.update(causal=rng.random() < 0.9, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                 softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.25)
    return c


def _lengths(case):
    """(cached tokens, new tokens) of every sequence: the case's own, whatever the seed of its values."""
    B, ctx, new = case["batch"], case["ctx"], case["new"]
    lens, news = [ctx] * B, [new] * B
    if case["ragged"]:
        r = random.Random(case["ragged"])
        for b in range(1, B):
            lens[b] = r.randint(max(1, ctx // 16), ctx)
            if new > 1:
                news[b] = lens[b] if case["new"] == case["ctx"] else r.randint(1, min(new, lens[b]))
        if B >= 4 and new == 1:
            lens[B - 1] = 0  # a slot of the batch that holds no sequence
    return lens, news


def _tile_bytes(D):
    return 16 * D + 96 * (D // 32)


def _offsets(D, dev):
    """Byte offsets inside a tile: codes [16 tokens, 2, G, 16], scales [16, 2, G], zeros [16, 2, G]."""
    G = D // 32
    tok = torch.arange(16, device=dev).view(16, 1, 1)
    g = torch.arange(G, device=dev).view(1, G, 1)
    b = torch.arange(16, device=dev).view(1, 1, 16)
    block = (tok // 8) * (4 * D)
    key = block + (tok % 8) * (D // 2) + ((b // 4) * G + g) * 4 + b % 4
    val = 8 * D + block + ((b // 2 * 4 + tok % 8 // 2) * G + g) * 4 + (tok % 2) * 2 + b % 2
    codes = torch.stack([key, val], 1)
    tok, g = tok[..., 0], g[..., 0]
    at = 16 * D
    scales = torch.stack([at + (tok * G + g) * 2, at + 32 * G + (tok // 2 * G + g) * 4 + tok % 2 * 2], 1)
    at += 64 * G
    zeros = torch.stack([at + tok * G + g, at + 16 * G + (tok // 2 * G + g) * 2 + tok % 2], 1)
    return codes, scales, zeros


def _quantise(x):
    """fp32 [..., D] -> codes u8 [..., G, 32], scales fp16 [..., G], zeros u8 [..., G]."""
    x = x.unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    s = ((hi - lo) * (1.0 / 15.0)).to(torch.float16)
    s32 = s.float()
    r = torch.where(s32 > 0, 1.0 / s32, torch.zeros_like(s32))
    z = torch.round(-lo * r).clamp(max=15)
    q = (torch.round(x * r) + z).clamp(0, 15)
    return q.to(torch.uint8), s[..., 0], z[..., 0].to(torch.uint8)


def _tables(rotary, rows, dev):
    if not rotary:
        return None, None
    freq = 500000.0 ** (-torch.arange(0, rotary, 2, device=dev, dtype=torch.float64) / rotary)
    ang = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _like_activations(shape, gen, dev, dt, spread):
    """Gaussian with a few loud features, as projections of trained models give."""
    x = torch.randn(shape, generator=gen, device=dev)
    loud = 1 + spread * (torch.rand(shape[-2:], generator=gen, device=dev) > 0.97)
    return (x * loud).to(dt)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    D, Hkv, Hq, P = case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    dt = _DTYPES[case["dtype"]]
    lens, news = _lengths(case)
    B, T = len(lens), sum(news)
    counts = [-(-n // P) for n in lens]
    width, pages = max(1, max(counts)), sum(counts) + 3
    perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    count = torch.tensor(counts, device=dev)
    col = torch.arange(width, device=dev)
    flat = (torch.cumsum(count, 0) - count)[:, None] + col
    tables = torch.where(col < count[:, None], perm[flat.clamp(max=pages - 1)], -1).to(torch.int32)
    seq_lens = torch.tensor(lens, device=dev, dtype=torch.int32)
    uniform = len(set(news)) == 1
    cu = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), device=dev, dtype=torch.int32)
    pool = torch.zeros(pages, Hkv, P // 16, _tile_bytes(D), dtype=torch.uint8, device=dev)
    st = dict(case=case, pool=pool, tables=tables, spare=perm[-1], seq_lens=seq_lens, cu=cu, news=torch.tensor(news, device=dev),
              T=T, max_new=max(news), max_len=max(lens), offsets=_offsets(D, dev), dt=dt)
    if case["op"] == "append":
        qkv = _like_activations((T, Hq + 2 * Hkv, D), gen, dev, dt, 8.0)
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        st["cos"], st["sin"] = _tables(case["rotary"], max(1, max(lens)), dev)
    else:
        codes, scales, zeros = st["offsets"]
        step = max(1, 40_000_000 // (Hkv * P * D))
        for p in range(0, pages, step):  # a full cache, page by page
            n = min(step, pages - p)
            for kv, spread in ((0, 6.0), (1, 2.0)):
                x = _like_activations((n, P // 16, 16, Hkv, D), gen, dev, torch.float32, spread)
                q, s, z = _quantise(x.permute(0, 3, 1, 2, 4))
                tile = pool[p:p + n]
                tile[..., codes[:, kv]] = q[..., 0::2] | (q[..., 1::2] << 4)
                b = s.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
                tile[..., scales[:, kv]], tile[..., scales[:, kv] + 1] = b[..., 0], b[..., 1]
                tile[..., zeros[:, kv]] = z
        st["q"] = _like_activations((T, Hq, D), gen, dev, dt, 3.0)
        st["slopes"] = None
        if case["alibi"]:
            st["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device=dev, dtype=torch.float32) / Hq)
    if own:
        from spectra_b200 import paged

        st["cache"] = paged.PagedKVCache.from_pool(pool, head_dim=D)
        st["batch"] = paged.TokenBatch(tables, seq_lens, cu_q=None if uniform else cu, q_len=news[0] if uniform else None,
                                       total=T, max_q=max(news), max_len=max(lens))
    return st


def _places(st):
    """Of every new token: its sequence and its position (negative: padding)."""
    seq = torch.repeat_interleave(torch.arange(len(st["news"]), device=st["news"].device), st["news"], output_size=st["T"])
    i = torch.arange(st["T"], device=seq.device) - st["cu"].long()[seq]
    return seq, st["seq_lens"].long()[seq] - st["news"][seq] + i


def _rotated(x, cos, sin, interleaved):
    x = x.float()
    if cos is None:
        return x
    rot = 2 * cos.shape[-1]
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _values(tiles, offsets):
    """Bytes [..., tile_bytes] -> fp32 [..., 16 tokens, 2, D]."""
    codes, scales, zeros = offsets
    b = tiles[..., codes]
    q = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    s = torch.stack([tiles[..., scales], tiles[..., scales + 1]], -1).view(torch.float16).float()
    z = tiles[..., zeros].float()[..., None]
    return ((q.float() - z) * s).flatten(-2)


def _run_append(st):
    c, pool = st["case"], st["pool"]
    P = c["page"]
    codes, scales, zeros = st["offsets"]
    seq, pos = _places(st)
    real = (pos >= 0)[:, None, None]
    at = pos.clamp(min=0)
    cos, sin = (None, None) if st["cos"] is None else (st["cos"][at], st["sin"][at])
    q = torch.where(real, _rotated(st["q"], cos, sin, c["interleaved"]), 0.0).to(st["dt"])
    k = _rotated(st["k"], cos, sin, c["interleaved"])
    code, s, z = _quantise(torch.stack([k, st["v"].float()], 2))  # [T, Hkv, 2, G, 32]
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    page = torch.where(pos >= 0, st["tables"][seq, at // P], st["spare"]).long()  # padding goes to an unused page
    rows = pool.view(-1)
    stride = pool.stride()
    base = page * stride[0] + at % P // 16 * stride[2]
    base = base[:, None] + torch.arange(c["kv_heads"], device=pool.device) * stride[1]
    token = at % 16
    to_code = base[:, :, None, None, None] + codes[token][:, None]
    to_scale = base[:, :, None, None] + scales[token][:, None]
    to_zero = base[:, :, None, None] + zeros[token][:, None]
    b = s.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
    rows[to_code], rows[to_zero] = packed, z
    rows[to_scale], rows[to_scale + 1] = b[..., 0], b[..., 1]
    # what the cache now holds of the new tokens
    b = rows[to_code]
    code = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()
    s = torch.stack([rows[to_scale], rows[to_scale + 1]], -1).view(torch.float16).float()
    kv = (code - rows[to_zero].float()[..., None]) * s
    kv = torch.where(real[..., None], kv.flatten(-2), 0.0).to(st["dt"])
    return {"q": q, "keys": kv[:, :, 0], "values": kv[:, :, 1]}


def _run_attend(st):
    c, pool, dev = st["case"], st["pool"], st["pool"].device
    B, Hq, Hkv, D, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    r = Hq // Hkv
    tiles = -(-max(1, st["max_len"]) // 16)
    t = torch.arange(tiles, device=dev)
    page = st["tables"][:, t * 16 // P].long().clamp(min=0)  # [B, tiles]
    kv = _values(pool[page, :, t % (P // 16)], st["offsets"])  # [B, tiles, Hkv, 16, 2, D]
    kv = kv.permute(4, 0, 2, 1, 3, 5).flatten(3, 4)  # [2, B, Hkv, L, D]
    L, N = tiles * 16, st["max_new"]
    seq, pos = _places(st)
    i = torch.arange(st["T"], device=dev) - st["cu"].long()[seq]
    q = torch.zeros(B, N, Hq, D, device=dev)
    q[seq, i] = st["q"].float()
    q = q.view(B, N, Hkv, r, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, r * N, D)
    s = (q @ kv[0].transpose(-1, -2)).view(B, Hkv, r, N, L) * (D ** -0.5)
    del q
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    n = torch.arange(L, device=dev)
    p = (st["seq_lens"].long() - st["news"])[:, None] + torch.arange(N, device=dev)  # [B, N]
    away = n - p[..., None]
    if c["alibi"]:
        s = s + st["slopes"].view(1, Hkv, r, 1, 1) * away[:, None, None]
    see = (n < st["seq_lens"][:, None])[:, None] & (p >= 0)[..., None]
    if c["causal"]:
        see = see & (away <= 0)
    if c["window"]:
        see = see & (away > -c["window"])
    s = torch.where(see[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = s.sum(-1, keepdim=True)
    o = (s.view(B, Hkv, r * N, L) @ kv[1]).view(B, Hkv, r, N, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)[seq, i].to(st["dt"])


def run(st):
    c = st["case"]
    if not own:
        return _run_append(st) if c["op"] == "append" else _run_attend(st)
    from spectra_b200 import paged

    if c["op"] == "append":
        q = paged.paged_kv_append(st["cache"], st["batch"], st["k"], st["v"], q=st["q"], cos=st["cos"], sin=st["sin"],
                                  interleaved=c["interleaved"])
        k, v = paged.paged_kv_read(st["cache"], st["batch"], dtype=st["dt"])
        return {"q": q, "keys": k, "values": v}
    return paged.paged_attention(st["q"], st["cache"], st["batch"], causal=c["causal"], window=c["window"],
                                 softcap=c["softcap"], alibi_slopes=st["slopes"])


def _visible(case):
    """Of every sequence: keys that some query sees, and pairs of a query and a key."""
    out = []
    for n, new in zip(*_lengths(case)):
        pairs, first, last = 0, n, -1
        for p in range(n - new, n):
            if p < 0:
                continue
            hi = p if case["causal"] else n - 1
            lo = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs, first, last = pairs + max(0, hi - lo + 1), min(first, lo), max(last, hi)
        out.append((max(0, last - first + 1), pairs))
    return out


def work(case):
    D, Hkv, Hq = case["head_dim"], case["kv_heads"], case["heads"]
    token = Hkv * (D + 6 * (D // 32))  # keys and values of one token, as held
    T = sum(_lengths(case)[1])
    if case["op"] == "append":
        move = 2 * Hq * D * 2 + 2 * Hkv * D * 2 + token + 4 * case["rotary"]  # rotate and append
        back = token + 2 * Hkv * D * 2  # read back
        return {"bytes": T * (move + back), "flops": T * (3 * Hq * case["rotary"] + Hkv * (3 * case["rotary"] + 8 * D))}
    vis = _visible(case)
    return {"bytes": sum(v[0] for v in vis) * token + 2 * T * Hq * D * 2, "flops": 4 * D * Hq * sum(v[1] for v in vis)}


def exact(case, seed):
    """64-bit results, one sequence and one head at a time."""
    st = prepare(case, seed)
    dev, f64 = st["pool"].device, torch.float64
    D, Hkv, Hq, P = case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    lens, news = _lengths(case)
    if case["op"] == "append":
        q, k, v = (st[x].to(f64) for x in "qkv")
        rot, base = case["rotary"], 0
        dead = torch.zeros(q.shape[0], dtype=torch.bool, device=dev)
        for n, new in zip(lens, news):
            for x in (q, k):
                if n < new:  # (padding: one token, no sequence)
                    dead[base:base + new - n] = True
                elif rot:
                    c, s = st["cos"][n - new:n].to(f64)[:, None], st["sin"][n - new:n].to(f64)[:, None]
                    lo = torch.arange(0, rot, 2, device=dev) if case["interleaved"] else torch.arange(rot // 2, device=dev)
                    hi = lo + 1 if case["interleaved"] else lo + rot // 2
                    row = x[base:base + new]
                    a, b = row[..., lo], row[..., hi]
                    row[..., lo], row[..., hi] = a * c - b * s, a * s + b * c
            base += new

        def held(x):
            g = x.reshape(x.shape[0], Hkv, D // 32, 32)
            low, high = g.min(-1, keepdim=True)[0].clamp(max=0), g.max(-1, keepdim=True)[0].clamp(min=0)
            s = ((high - low) / 15).to(torch.float16).to(f64)
            z = torch.where(s > 0, torch.round(-low / s), 0.0).clamp(0, 15)
            code = torch.where(s > 0, torch.round(g / s) + z, 0.0).clamp(0, 15)
            return ((code - z) * s).reshape(x.shape)

        res = {"q": q, "keys": held(k), "values": held(v)}
        for x in res.values():
            x[dead] = 0
        return res
    G, out, base = D // 32, torch.zeros(st["T"], Hq, D, dtype=f64, device=dev), 0
    for b, (n, new) in enumerate(zip(lens, news)):
        if n == 0:
            base += new
            continue
        pages = st["tables"][b, :-(-n // P)].long()
        pos = torch.arange(n - new, n, device=dev)[:, None]
        key = torch.arange(n, device=dev)[None]
        see = (pos >= 0) & (key < n)
        if case["causal"]:
            see = see & (key <= pos)
        if case["window"]:
            see = see & (key > pos - case["window"])
        for h in range(Hkv):
            raw = st["pool"][pages, h].reshape(-1, _tile_bytes(D))
            words = raw[:, :8 * D].reshape(-1, 8, 4, G, 4)  # 8-token blocks: token, word, group, byte
            kc = torch.stack([words & 15, words >> 4], -1).permute(0, 1, 3, 2, 4, 5).reshape(-1, G, 32)
            words = raw[:, 8 * D:16 * D].reshape(-1, 8, 4, G, 2, 2)  # lane, pair, group, token of the pair, byte
            vc = torch.stack([words & 15, words >> 4], -1).permute(0, 2, 4, 3, 1, 5, 6).reshape(-1, G, 32)
            half = raw[:, 16 * D:16 * D + 64 * G].contiguous().view(torch.float16).to(f64)
            zero = raw[:, 16 * D + 64 * G:].to(f64)
            ks, kz = half[:, :16 * G].reshape(-1, G, 1), zero[:, :16 * G].reshape(-1, G, 1)
            vs = half[:, 16 * G:].reshape(-1, G, 2).transpose(1, 2).reshape(-1, G, 1)
            vz = zero[:, 16 * G:].reshape(-1, G, 2).transpose(1, 2).reshape(-1, G, 1)
            K = ((kc.to(f64) - kz) * ks).reshape(-1, D)[:n]
            V = ((vc.to(f64) - vz) * vs).reshape(-1, D)[:n]
            for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                s = st["q"][base:base + new, j].to(f64) @ K.T / math.sqrt(D)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                if case["alibi"]:
                    s = s - st["slopes"][j].to(f64) * (pos - key)
                s = s.masked_fill(~see, -math.inf)
                w = torch.softmax(s, -1).nan_to_num(0.0)  # (a row that sees nothing: zeros)
                out[base:base + new, j] = w @ V
        base += new
    return out
