"""Performance cases of a long-context serving step's operators: the block index of a paged cache, the choice of
blocks and the attention over them, the append with several position axes, and rules on logits.

Each case is one pass through one operator (``sparse``: the choice and the attention that reads it), from single
tokens to long prompts.  ``run`` computes it with elementary torch operations, or, where ``own`` is set, with
``spectra_b200.paged`` and ``spectra_b200.logits``.

A cache is one byte tensor [pages, kv_heads, page / 16, tile_bytes].  A tile holds 16 tokens of one head, D = 32 G
features each:
  key codes    [2 blocks of 8 tokens][8 tokens][4 words c][G]: word c of group g holds features 8c..8c+7 of the group
  value codes  [2 blocks][8 lanes l][4 token pairs][G]: features 4l..4l+3 of the even token in the low half of the word,
               of the odd token in the high half
  key scales   fp16 [16][G],   value scales  fp16 [8 token pairs][G][2]
  key zeros    u8   [16][G],   value zeros   u8   [8 token pairs][G][2]
and a code q stands for (q - zero) * scale.

A block index holds, of every block of ``block`` tokens of a page and every head, the largest and the smallest value
of each key feature, rounded outwards to integers of 8 bits times one power of two.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


def _paged(name, op, **kw):
    c = dict(name=name, op=op, dtype="bf16", heads=32, kv_heads=8, head_dim=128, page=64, block=64, batch=1, ctx=1024,
             new=1, ragged=0, count=0, first=1, last=1, softcap=0.0, alibi=False, rotary=0, interleaved=False, order="runs")
    c.update(kw)
    return c


def _logits(name, **kw):
    c = dict(name=name, op="logits", dtype="bf16", rows=1, vocab=128256, history=1024, ragged=0, penalties=True, bias=0,
             mask="none")
    c.update(kw)
    return c


def listed():
    return [
        # a decode step of a busy server: in some of 128 sequences the new token is a block's last one
        _paged("index-128-sequences", "index", batch=128, ctx=1000, ragged=1),
        # ragged prompts that have just been appended
        _paged("index-prompts", "index", batch=6, ctx=16384, new=16384, ragged=2),
        # one token of one long conversation, 8B-shaped layer: 2048 blocks to choose 32 from
        _paged("sparse-one-131072", "sparse", ctx=131072, count=32),
        # decode step of a busy server on a 70B-shaped layer, long sequences
        _paged("sparse-64-sequences", "sparse", heads=64, batch=64, ctx=16384, ragged=3, count=32, last=2),
        # checking up to five drafted tokens of 16 sequences on a 1B-shaped layer, fp16, a score cap, small blocks
        _paged("sparse-verify-cap-fp16", "sparse", dtype="fp16", head_dim=64, page=32, block=32, batch=16, ctx=6001, new=5,
               ragged=4, count=24, first=2, last=3, softcap=50.0),
        # a chunk of new tokens of a long prompt, every token with its own choice
        _paged("sparse-chunk-512", "sparse", ctx=32768, new=512, count=16),
        # one token of 16 conversations with images
        _paged("append-axes-16-sequences", "append", batch=16, ctx=4096, ragged=5, rotary=128),
        # ragged prompts with images, fp16, axes taken by turns, a part of the head rotated
        _paged("append-axes-images-fp16", "append", dtype="fp16", heads=16, kv_heads=4, head_dim=96, page=32, batch=5,
               ctx=2049, new=2049, ragged=6, rotary=48, order="turns"),
        # a video's frames on a 70B-shaped layer
        _paged("append-axes-video", "append", heads=64, ctx=16384, new=16384, rotary=128),
        # the next token of one conversation
        _logits("logits-one", history=1281),
        # a decode step of a busy server: penalties, biases and a grammar each
        _logits("logits-64-rows", rows=64, history=8192, ragged=7, bias=300, mask="mixed"),
        # drafted tokens of many sequences, odd vocabulary, fp16, a grammar that leaves little
        _logits("logits-333-rows-fp16", dtype="fp16", rows=333, vocab=50001, history=2001, ragged=8, bias=17, mask="tight"),
    ]


_HEADS = [(32, 8, 64), (32, 8, 128), (64, 8, 128), (4, 2, 64), (16, 16, 64), (32, 32, 128), (16, 4, 96), (8, 4, 256),
          (8, 1, 32), (40, 8, 128), (12, 1, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["index", "sparse", "sparse", "append", "logits"])
    if op == "logits":
        rows, vocab = _log(rng, 1, 512), rng.choice([128256, _log(rng, 1000, 200000), _log(rng, 1000, 200000)])
        rows = max(1, min(rows, 64 * 128256 // vocab))
        history = min(_log(rng, 1, 32768), 64 * 8192 // rows)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=rows, vocab=vocab, history=history,
                    ragged=rng.randrange(1, 1000), penalties=rng.random() < 0.8, bias=rng.choice([0, _log(rng, 1, 512)]),
                    mask=rng.choice(["none", "mixed", "tight"]))
    heads, kv_heads, dim = rng.choice(_HEADS)
    page = rng.choice([32, 64, 128, 256])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), heads=heads, kv_heads=kv_heads, head_dim=dim, page=page,
             block=rng.choice([b for b in (32, 64, 128) if b <= page]), ragged=rng.randrange(1, 1000), count=0, first=1,
             last=1, softcap=0.0, alibi=False, rotary=0, interleaved=False, order="runs")
    form = rng.choice(["one", "one", "few", "many"])
    if form == "one":
        batch, ctx, new = _log(rng, 1, 200), _log(rng, 16, 131072), 1
    elif form == "few":
        batch, ctx, new = _log(rng, 1, 32), _log(rng, 32, 65536), rng.randrange(2, 9)
    else:
        batch, new = _log(rng, 1, 8), _log(rng, 64, 512 if op == "sparse" else 8192)
        ctx = new if op != "sparse" and rng.random() < 0.6 else new + _log(rng, 1, 32768)
    if op == "index" and form != "many":  # (only the last blocks are read, whatever the length)
        ctx = max(new, min(ctx, 1000))
    room = 75_000_000 if op == "index" else 200_000_000  # cached values
    ctx = max(new, min(ctx, room // (batch * kv_heads * dim)))
    while batch > 1 and batch * kv_heads * dim * ctx > room:
        batch //= 2
    if op == "append":
        while batch > 1 and batch * new * (heads + kv_heads) * dim > 16384 * 72 * 128:
            batch //= 2
        new = max(1, min(new, 16384 * 72 * 128 // ((heads + kv_heads) * dim)))
        c.update(rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, order=rng.choice(["runs", "turns"]))
    if op == "sparse":
        block = c["block"]
        c.update(first=rng.randrange(0, 3), last=rng.randrange(1, 4), softcap=rng.choice([0.0, 0.0, 30.0]),
                 alibi=rng.random() < 0.2)
        count = max(6, min(_log(rng, 6, 96), 4096 // block))
        each = heads * dim * (count * block + ctx // block)  # products of one token
        while batch > 1 and batch * new * each > 512 * 32 * 128 * 1500:
            batch //= 2
        new = max(1, min(new, 512 * 32 * 128 * 1500 // (batch * each)))
        c.update(count=count)
    c.update(batch=batch, ctx=ctx, new=new)
    return c


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """(cached tokens, new tokens) of every sequence: the case's own, whatever the seed of its values."""
    B, ctx, new = case["batch"], case["ctx"], case["new"]
    lens, news = [ctx] * B, [new] * B
    if case["ragged"]:
        r = random.Random(case["ragged"])
        for b in range(1, B):
            lens[b] = r.randint(max(1, ctx // 16), ctx)
            if case["op"] == "index" and new == 1 and r.random() < 0.3:  # more full blocks than chance gives
                lens[b] = max(lens[b] // case["block"], 1) * case["block"]
            if new > 1:
                news[b] = lens[b] if new == ctx else r.randint(1, min(new, lens[b]))
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


def _like_activations(shape, gen, dev, dt, spread):
    """Gaussian with a few loud features, as projections of trained models give."""
    x = torch.randn(shape, generator=gen, device=dev)
    loud = 1 + spread * (torch.rand(shape[-2:], generator=gen, device=dev) > 0.97)
    return (x * loud).to(dt)


def _pair_axes(half, order):
    """Axis (time, height, width) of each pair of the rotated part."""
    if order == "turns":
        return [i % 3 for i in range(half)]
    a = half // 4
    b = (half - a) // 2
    return [0] * a + [1] * b + [2] * (half - a - b)


def _axis_positions(lens, news, seed):
    """Positions [3, T] as a preprocessor gives them: runs of text count up on all axes, images and frames spread out."""
    r, cols = random.Random(seed), []
    for n, new in zip(lens, news):
        if new == 1:
            cols.append([[max(0, n - 1 - r.randint(0, n // 2))] * 3] if n else [[0] * 3])
            continue
        row, at = [], 0
        while len(row) < new:
            if r.random() < 0.5:
                for _ in range(r.randint(1, 200)):
                    row.append([at] * 3)
                    at += 1
            else:
                frames, h, w = r.randint(1, 8), r.randint(4, 24), r.randint(4, 24)
                row += [[at + f, at + y, at + x] for f in range(frames) for y in range(h) for x in range(w)]
                at += max(frames, h, w)
        cols.append(row[:new])
    return [[p[a] for row in cols for p in row] for a in range(3)]


def _prepare_paged(case, seed):
    dev = torch.device(_DEV)
    gen = torch.Generator(device=dev).manual_seed(seed)
    D, Hkv, Hq, P, BS = case["head_dim"], case["kv_heads"], case["heads"], case["page"], case["block"]
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
    codes, scales, zeros = st["offsets"]
    if case["op"] == "append":
        qkv = _like_activations((T, Hq + 2 * Hkv, D), gen, dev, dt, 8.0)
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        rotary, rows = case["rotary"], max(16, max(lens))
        freq = 500000.0 ** (-torch.arange(0, rotary, 2, device=dev, dtype=torch.float64) / rotary)
        ang = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["positions"] = torch.tensor(_axis_positions(lens, news, seed), dtype=torch.int32, device=dev)
        st["pair_axes"] = torch.tensor(_pair_axes(rotary // 2, case["order"]), device=dev)
    else:
        step = max(1, 40_000_000 // (Hkv * P * D))
        for p in range(0, pages, step):  # a full cache, page by page; keys drift from block to block
            n = min(step, pages - p)
            for kv, spread in ((0, 6.0), (1, 2.0)):
                x = _like_activations((n, P // 16, 16, Hkv, D), gen, dev, torch.float32, spread)
                if kv == 0:
                    drift = torch.randn(n, P // BS, 1, Hkv, D, generator=gen, device=dev)
                    x = (x.view(n, P // BS, BS, Hkv, D) + drift).view(x.shape)
                q, s, z = _quantise(x.permute(0, 3, 1, 2, 4))
                tile = pool[p:p + n]
                tile[..., codes[:, kv]] = q[..., 0::2] | (q[..., 1::2] << 4)
                b = s.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
                tile[..., scales[:, kv]], tile[..., scales[:, kv] + 1] = b[..., 0], b[..., 1]
                tile[..., zeros[:, kv]] = z
        st["codes"] = torch.zeros(pages, Hkv, P // BS, 2, D, dtype=torch.int8, device=dev)
        st["scales"] = torch.zeros(pages, Hkv, P // BS, dtype=torch.float32, device=dev)
        if case["op"] == "sparse":
            st["q"] = _like_activations((T, Hq, D), gen, dev, dt, 3.0)
            st["slopes"] = None
            if case["alibi"]:
                st["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device=dev, dtype=torch.float32) / Hq)
            for p in range(0, pages, step):  # the index that the program has kept so far
                st["codes"][p:p + step], st["scales"][p:p + step] = _bounds(_keys(pool[p:p + step], st["offsets"]), BS)
    if own:
        from spectra_b200 import paged

        st["cache"] = paged.PagedKVCache.from_pool(pool, head_dim=D)
        st["batch"] = paged.TokenBatch(tables, seq_lens, cu_q=None if uniform else cu, q_len=news[0] if uniform else None,
                                       total=T, max_q=max(news), max_len=max(lens))
        if case["op"] == "append":
            st["axes"] = paged.RotaryAxes(st["pair_axes"].tolist())
        else:
            st["index"] = paged.BlockIndex.from_buffers(st["cache"], st["codes"], st["scales"])
    return st


def _prepare_logits(case, seed):
    dev = torch.device(_DEV)
    gen = torch.Generator(device=dev).manual_seed(seed)
    M, V, H = case["rows"], case["vocab"], case["history"]
    r = random.Random(case["ragged"])
    logits = (2.5 * torch.randn(M, V, generator=gen, device=dev)).to(_DTYPES[case["dtype"]])
    st = dict(case=case, logits=logits, ids=None, lengths=None, prompt=None, repetition=None, frequency=None, presence=None,
              bias_ids=None, bias=None, allowed=None)
    if case["penalties"]:
        lengths = [H] + [r.randint(0, H) if case["ragged"] else H for _ in range(M - 1)]
        # text repeats itself: most ids are among the few frequent ones
        u = torch.rand(M, H, generator=gen, device=dev, dtype=torch.float64)
        st["ids"] = (V * u ** 4).long().clamp(max=V - 1).to(torch.int32)
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        st["prompt"] = torch.tensor([r.randint(0, n) for n in lengths], dtype=torch.int32, device=dev)
        pick = lambda *c: torch.tensor([r.choice(c) for _ in range(M)], dtype=torch.float32, device=dev)  # noqa: E731
        st["repetition"], st["frequency"], st["presence"] = pick(1.0, 1.1, 1.3), pick(0.0, 0.25, 0.7), pick(0.0, 0.5)
    if case["bias"]:
        st["bias_ids"] = torch.randint(0, V, (M, case["bias"]), generator=gen, device=dev).to(torch.int32)
        st["bias_ids"][:, 1::7] = -1  # rows with fewer biases
        st["bias"] = 4.0 * torch.randn(M, case["bias"], generator=gen, device=dev)
    if case["mask"] != "none":
        words = -(-V // 32)
        if case["mask"] == "mixed":  # rows without a grammar, rows in the middle of a free string
            word = torch.randint(-2**31, 2**31, (M, words), generator=gen, device=dev).to(torch.int32)
            word[::2] = -1
        else:  # a few tokens can follow, in one row none
            word = torch.randint(-2**31, 2**31, (M, words), generator=gen, device=dev).to(torch.int32)
            word[torch.rand(M, words, generator=gen, device=dev) > 9 / words] = 0
            word[M // 2] = 0
        st["allowed"] = word
    if own:
        from spectra_b200 import logits as rules

        st["rules"] = rules.LogitRules(ids=st["ids"], lengths=st["lengths"], prompt_lengths=st["prompt"],
                                       repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                                       bias_ids=st["bias_ids"], bias=st["bias"], allowed=st["allowed"])
    return st


def prepare(case, seed):
    return _prepare_logits(case, seed) if case["op"] == "logits" else _prepare_paged(case, seed)


# ------------------------------------------------------------------ the plain forms

def _values(tiles, offsets):
    """Bytes [..., tile_bytes] -> fp32 [..., 16 tokens, 2, D]."""
    codes, scales, zeros = offsets
    b = tiles[..., codes]
    q = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    s = torch.stack([tiles[..., scales], tiles[..., scales + 1]], -1).view(torch.float16).float()
    z = tiles[..., zeros].float()[..., None]
    return ((q.float() - z) * s).flatten(-2)


def _keys(pages, offsets):
    """Pages [n, H, page / 16, tile_bytes] -> fp32 keys [n, H, page, D]."""
    codes, scales, zeros = offsets
    return _values(pages, (codes[:, :1], scales[:, :1], zeros[:, :1]))[..., 0, :].flatten(2, 3)


def _power(most):
    """The least power of two (2^-126 at least) times 127 that reaches fp32 ``most``; 1 where it is 0."""
    m, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1; 127 = 0.9921875 2^7
    e = torch.where(m > 0.9921875, e - 6, e - 7).clamp(min=-126)
    return torch.where(most > 0, torch.ldexp(torch.ones_like(most), e), 1.0)


def _bounds(keys, block):
    """Keys [n, H, page, D] -> codes int8 [n, H, page / block, 2, D], scales fp32 [n, H, page / block]."""
    k = keys.unflatten(2, (-1, block))
    hi, lo = k.amax(3), k.amin(3)
    s = _power(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    return torch.stack([torch.ceil(hi / s[..., None]), torch.floor(lo / s[..., None])], 3).to(torch.int8), s


def _places(st):
    """Of every new token: its sequence and its position (negative: padding)."""
    seq = torch.repeat_interleave(torch.arange(len(st["news"]), device=st["news"].device), st["news"], output_size=st["T"])
    i = torch.arange(st["T"], device=seq.device) - st["cu"].long()[seq]
    return seq, st["seq_lens"].long()[seq] - st["news"][seq] + i


def _run_index(st):
    c, P, BS = st["case"], st["case"]["page"], st["case"]["block"]
    seq, pos = _places(st)
    # the blocks that a new token filled: where its page is, and which of the page's
    full = ((pos >= 0) & (pos % BS == BS - 1)).nonzero()[:, 0]
    seq, pos = seq[full], pos[full]
    page, part = st["tables"][seq, pos // P].long(), pos % P // BS
    step = max(1, 60_000_000 // (c["kv_heads"] * BS * c["head_dim"]))
    for i in range(0, len(page), step):
        at, of = page[i:i + step], part[i:i + step]
        tiles = of[:, None] * (BS // 16) + torch.arange(BS // 16, device=at.device)
        keys = _keys(st["pool"][at[:, None], :, tiles].transpose(1, 2), st["offsets"])
        codes, scales = _bounds(keys, BS)
        st["codes"][at, :, of], st["scales"][at, :, of] = codes[:, :, 0], scales[:, :, 0]
    return {"bounds": st["codes"].float() * st["scales"][..., None, None]}


def _run_sparse(st):
    c, pool, dev = st["case"], st["pool"], st["pool"].device
    Hq, Hkv, D, P, BS, K = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["block"], c["count"]
    r, T = Hq // Hkv, st["T"]
    NB = -(-max(1, st["max_len"]) // BS)
    seq, pos = _places(st)
    j = torch.arange(NB, device=dev)
    page, part = st["tables"][:, j * BS // P].long(), j % (P // BS)  # [B, NB]
    q = st["q"].float().view(T, Hkv, r, D)
    code = torch.round(q / _power(q.abs().amax(-1, keepdim=True)))
    blocks = torch.empty(T, Hkv, K, dtype=torch.int32, device=dev)
    out = torch.empty(T, Hq, D, dtype=st["dt"], device=dev)
    for b in range(len(st["news"])):
        at = st["cu"][b] + torch.arange(int(c["new"] if c["ragged"] == 0 else st["news"][b]), device=dev)
        p = pos[at]
        own_block = torch.div(p, BS, rounding_mode="floor")
        held = page[b] >= 0
        hi, lo = st["codes"][page[b].clamp(min=0), :, part].float().permute(2, 1, 0, 3)  # [2][Hkv, NB, D]
        x = code[at].permute(1, 0, 2, 3).flatten(1, 2)  # [Hkv, n r, D]
        s = x.clamp(min=0) @ hi.transpose(1, 2) + x.clamp(max=0) @ lo.transpose(1, 2)
        s = s.view(Hkv, len(at), r, NB).amax(2).transpose(0, 1) * st["scales"][page[b].clamp(min=0), :, part].T
        always = (j < c["first"]) | (j > own_block[:, None] - c["last"])
        s = torch.where(always[:, None], math.inf, s)
        s = torch.where(((j <= own_block[:, None]) & held)[:, None], s, -math.inf)  # [n, Hkv, NB]
        best, order = torch.sort(s, dim=-1, descending=True, stable=True)
        order = torch.where(best == -math.inf, NB, order)[..., :K].sort(-1)[0]
        order = torch.nn.functional.pad(order, (0, K - order.shape[-1]), value=NB)
        blocks[at] = torch.where(order < NB, order, -1).to(torch.int32)
        step = max(1, 40_000_000 // (Hkv * K * BS * D))
        for i in range(0, len(at), step):
            rows, sel = at[i:i + step], order[i:i + step]  # [n, Hkv, K]
            n = (sel[..., None] * BS + torch.arange(BS, device=dev)).flatten(2)  # positions [n, Hkv, K BS]
            tile = (sel[..., None] * (BS // 16) + torch.arange(BS // 16, device=dev)).flatten(2)
            where = st["tables"][b].long()[(tile * 16 // P).clamp(max=st["tables"].shape[1] - 1)].clamp(min=0)
            kv = _values(pool[where, torch.arange(Hkv, device=dev)[:, None], tile % (P // 16)], st["offsets"])
            kv = kv.flatten(2, 3)  # [n, Hkv, K BS, 2, D]
            w = (q[rows] @ kv[..., 0, :].transpose(-1, -2)) * D ** -0.5  # [n, Hkv, r, K BS]
            if c["softcap"]:
                w = c["softcap"] * torch.tanh(w / c["softcap"])
            away = n - pos[rows][:, None, None]
            if c["alibi"]:
                w = w + st["slopes"].view(Hkv, r, 1) * away[:, :, None]
            see = (away <= 0) & (sel < NB).repeat_interleave(BS, -1)
            w = torch.where(see[:, :, None], w, -math.inf)
            m = w.amax(-1, keepdim=True)
            w = torch.exp(w - torch.where(m == -math.inf, 0.0, m))
            total = w.sum(-1, keepdim=True)
            o = (w @ kv[..., 1, :]) / torch.where(total > 0, total, 1.0)
            out[rows] = o.flatten(1, 2).to(st["dt"])
    return {"blocks": blocks, "out": out}


def _run_append(st):
    c, pool = st["case"], st["pool"]
    P, rot = c["page"], c["rotary"]
    codes, scales, zeros = st["offsets"]
    seq, pos = _places(st)
    real = (pos >= 0)[:, None, None]
    at = pos.clamp(min=0)
    row = st["positions"].long()[st["pair_axes"]].T  # [T, pairs]
    cos, sin = (x.gather(0, row)[:, None] for x in (st["cos"], st["sin"]))

    def turned(x):
        x = x.float()
        part = x[..., :rot]
        a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else part.chunk(2, -1)
        u, w = a * cos - b * sin, b * cos + a * sin
        part = torch.stack([u, w], -1).flatten(-2) if c["interleaved"] else torch.cat([u, w], -1)
        return torch.cat([part, x[..., rot:]], -1)

    q = torch.where(real, turned(st["q"]), 0.0).to(st["dt"])
    code, s, z = _quantise(torch.stack([turned(st["k"]), st["v"].float()], 2))  # [T, Hkv, 2, G, 32]
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


def _run_logits(st):
    x = st["logits"].float()
    M, V = x.shape
    if st["ids"] is not None:
        i = torch.arange(st["ids"].shape[1], device=x.device)
        ids, held = st["ids"].long(), i < st["lengths"][:, None]
        new = held & (i >= st["prompt"][:, None])
        seen = torch.zeros(M, V, dtype=torch.int32, device=x.device).scatter_add_(1, ids, held.int())
        times = torch.zeros(M, V, dtype=torch.int32, device=x.device).scatter_add_(1, ids, new.int())
        r = st["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - st["frequency"][:, None] * times.float()
        x = x - torch.where(times > 0, st["presence"][:, None], 0.0)
    if st["bias_ids"] is not None:  # the last entry of an id counts
        n = st["bias_ids"].shape[1]
        which = torch.zeros(M, V + 1, dtype=torch.int64, device=x.device)
        ids = torch.where(st["bias_ids"] >= 0, st["bias_ids"].long(), V)
        which.scatter_reduce_(1, ids, torch.arange(1, n + 1, device=x.device).expand(M, n), "amax")
        x = x + torch.cat([torch.zeros(M, 1, device=x.device), st["bias"]], 1).gather(1, which[:, :V])
    ok = torch.ones(M, V, dtype=torch.bool, device=x.device)
    if st["allowed"] is not None:
        n = torch.arange(V, device=x.device)
        ok = (st["allowed"][:, n // 32] >> (n % 32)) & 1 > 0
        x = torch.where(ok, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    token = ((x == top) & ok).to(torch.int8).argmax(-1)  # (argmax of equal values: the first)
    return {"logits": x.to(st["logits"].dtype), "tokens": torch.where(ok.any(-1), token, -1)}


_PLAIN = {"index": _run_index, "sparse": _run_sparse, "append": _run_append, "logits": _run_logits}


def run(st):
    c = st["case"]
    if not own:
        return _PLAIN[c["op"]](st)
    if c["op"] == "logits":
        from spectra_b200 import logits

        x, tokens = logits.adjust_logits(st["logits"], st["rules"], with_tokens=True)
        return {"logits": x, "tokens": tokens}
    from spectra_b200 import paged

    if c["op"] == "index":
        paged.paged_index_update(st["index"], st["batch"])
        return {"bounds": st["codes"] * st["scales"][..., None, None]}
    if c["op"] == "append":
        q = paged.paged_kv_append(st["cache"], st["batch"], st["k"], st["v"], q=st["q"], cos=st["cos"], sin=st["sin"],
                                  interleaved=c["interleaved"], positions=st["positions"], axes=st["axes"])
        k, v = paged.paged_kv_read(st["cache"], st["batch"], dtype=st["dt"])
        return {"q": q, "keys": k, "values": v}
    blocks = paged.paged_select_blocks(st["q"], st["index"], st["batch"], c["count"], first=c["first"], last=c["last"])
    o = paged.paged_attention(st["q"], st["cache"], st["batch"], softcap=c["softcap"], alibi_slopes=st["slopes"],
                              blocks=blocks, block_size=c["block"])
    return {"blocks": blocks, "out": o}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "logits":
        size = 4 if case["dtype"] == "fp32" else 2
        M, V = case["rows"], case["vocab"]
        ids = M * case["history"] * 4 // (2 if case["ragged"] and M > 1 else 1) if case["penalties"] else 0
        mask = M * -(-V // 32) * 4 if case["mask"] != "none" else 0
        return {"bytes": 2 * M * V * size + ids + 8 * M * case["bias"] + mask + 8 * M, "flops": 2 * M * V}
    D, Hkv, Hq, BS = case["head_dim"], case["kv_heads"], case["heads"], case["block"]
    G = D // 32
    lens, news = _lengths(case)
    T = sum(news)
    token = Hkv * (D + 6 * G)  # keys and values of one token, as held
    if case["op"] == "append":
        move = 2 * Hq * D * 2 + 2 * Hkv * D * 2 + token + 4 * case["rotary"] + 12
        back = token + 2 * Hkv * D * 2
        return {"bytes": T * (move + back), "flops": T * (3 * Hq * case["rotary"] + Hkv * (3 * case["rotary"] + 8 * D))}
    if case["op"] == "index":
        full = sum(n // BS - max(0, n - new) // BS for n, new in zip(lens, news))
        pages = sum(-(-n // case["page"]) for n in lens) + 3
        values = pages * (case["page"] // BS) * Hkv * (2 * D * 5 + 4)  # the bounds read and returned as numbers
        return {"bytes": full * Hkv * (BS * (D // 2 + 3 * G) + 2 * D + 4) + values, "flops": full * Hkv * BS * 4 * D}
    moved, ops = 2 * T * Hq * D * 2 + 2 * T * Hkv * case["count"] * 4, 0
    for n, new in zip(lens, news):
        scored, keys = 0, 0
        for p in range(max(0, n - new), n):
            own_block = p // BS
            if own_block + 1 > case["count"]:
                scored += own_block + 1 - case["first"] - case["last"]
            keys += min(own_block, case["count"] - 1) * BS + p % BS + 1
        last = max(0, n - 1) // BS
        moved += (Hkv * last * (2 * D + 4) if scored else 0) + min(keys, n) * token
        ops += 4 * D * Hq * (scored + keys)
    return {"bytes": moved, "flops": ops}


# ------------------------------------------------------------------ 64 bits, from the definitions

def _unpacked(raw, D):
    """Tiles [n, tile_bytes] of one head -> fp64 keys and values [16 n, D]."""
    G, f64 = D // 32, torch.float64
    words = raw[:, :8 * D].reshape(-1, 8, 4, G, 4)  # 8-token blocks: token, word, group, byte
    kc = torch.stack([words & 15, words >> 4], -1).permute(0, 1, 3, 2, 4, 5).reshape(-1, G, 32)
    words = raw[:, 8 * D:16 * D].reshape(-1, 8, 4, G, 2, 2)  # lane, pair, group, token of the pair, byte
    vc = torch.stack([words & 15, words >> 4], -1).permute(0, 2, 4, 3, 1, 5, 6).reshape(-1, G, 32)
    half = raw[:, 16 * D:16 * D + 64 * G].contiguous().view(torch.float16).to(f64)
    zero = raw[:, 16 * D + 64 * G:].to(f64)
    ks, kz = half[:, :16 * G].reshape(-1, G, 1), zero[:, :16 * G].reshape(-1, G, 1)
    vs = half[:, 16 * G:].reshape(-1, G, 2).transpose(1, 2).reshape(-1, G, 1)
    vz = zero[:, 16 * G:].reshape(-1, G, 2).transpose(1, 2).reshape(-1, G, 1)
    return ((kc.to(f64) - kz) * ks).reshape(-1, D), ((vc.to(f64) - vz) * vs).reshape(-1, D)


def _step64(most):
    """fp64: the power of two s with 63.5 s < most <= 127 s; 1 for 0."""
    s = torch.exp2(torch.ceil(torch.log2(most.clamp(min=1e-300) / 127.0)))
    s = torch.where(most > 127 * s, 2 * s, s)
    return torch.where(most > 0, torch.where(most <= 63.5 * s, s / 2, s), 1.0)


def _exact_index(case, st, lens, news):
    D, P, BS, dev = case["head_dim"], case["page"], case["block"], st["pool"].device
    out = torch.zeros(st["codes"].shape, dtype=torch.float64, device=dev)
    for b, (n, new) in enumerate(zip(lens, news)):
        if n // BS == max(0, n - new) // BS:
            continue
        pages = st["tables"][b, :-(-n // P)].long()
        done = torch.arange(max(0, n - new) // BS, n // BS, device=dev)
        for h in range(case["kv_heads"]):
            K, _ = _unpacked(st["pool"][pages, h].reshape(-1, _tile_bytes(D)), D)
            g = K[:len(K) // BS * BS].reshape(-1, BS, D)[done]
            both = torch.stack([g.max(1)[0], g.min(1)[0]], 1)
            s = _step64(both.abs().flatten(1).max(1)[0])[:, None]
            both = torch.stack([torch.ceil(both[:, 0] / s), torch.floor(both[:, 1] / s)], 1) * s[..., None]
            out[pages[done * BS // P], h, done % (P // BS)] = both
    return {"bounds": out}


def _exact_sparse(case, st, lens, news):
    D, Hkv, Hq, P, BS, K = (case[x] for x in ("head_dim", "kv_heads", "heads", "page", "block", "count"))
    r, dev, f64 = Hq // Hkv, st["pool"].device, torch.float64
    if sum(news) * Hkv > 8000:
        return None
    blocks = torch.full((st["T"], Hkv, K), -1, dtype=torch.int32, device=dev)
    out, base = torch.zeros(st["T"], Hq, D, dtype=f64, device=dev), 0
    for b, (n, new) in enumerate(zip(lens, news)):
        pages = st["tables"][b, :-(-n // P)].long()
        for h in range(Hkv if n else 0):
            keys, vals = _unpacked(st["pool"][pages, h].reshape(-1, _tile_bytes(D)), D)
            full = n // BS
            g = keys[:full * BS].reshape(full, BS, D)
            up = g.max(1)[0] if full else keys[:0]
            down = g.min(1)[0] if full else keys[:0]
            s = _step64(torch.maximum(up.abs(), down.abs()).max(1)[0])[:, None] if full else up[:, :1]
            up, down = torch.ceil(up / s) * s, torch.floor(down / s) * s  # [full, D]
            for t in range(base, base + new):
                p = n - new + t - base
                if p < 0:
                    continue
                q = st["q"][t, h * r:(h + 1) * r].to(f64)
                last = p // BS
                must = set(range(min(case["first"], last + 1))) | set(range(max(0, last + 1 - case["last"]), last + 1))
                rest = [j for j in range(last + 1) if j not in must]
                free = max(0, K - len(must))
                if len(rest) > free:
                    c = torch.round(q / _step64(q.abs().max(1)[0])[:, None])[:, None]
                    lo, hi = rest[0], rest[-1] + 1
                    score = torch.where(c > 0, c * up[lo:hi], c * down[lo:hi]).sum(-1).max(0)[0]
                    rest = (torch.sort(score, dim=0, descending=True, stable=True)[1][:free] + lo).tolist()
                pick = torch.tensor(sorted(must | set(rest)), device=dev)
                blocks[t, h, :len(pick)] = pick.to(torch.int32)
                at = (pick[:, None] * BS + torch.arange(BS, device=dev)).flatten()
                at = at[at <= p]
                w = q @ keys[at].T / math.sqrt(D)
                if case["softcap"]:
                    w = case["softcap"] * torch.tanh(w / case["softcap"])
                if case["alibi"]:
                    w = w + st["slopes"][h * r:(h + 1) * r, None].to(f64) * (at - p)
                out[t, h * r:(h + 1) * r] = torch.softmax(w, -1) @ vals[at]
        base += new
    return {"blocks": blocks, "out": out}


def _exact_append(case, st, lens, news):
    D, Hkv, rot, dev, f64 = case["head_dim"], case["kv_heads"], case["rotary"], st["pool"].device, torch.float64
    q, k, v = (st[x].to(f64) for x in "qkv")
    dead, base = torch.zeros(st["T"], dtype=torch.bool, device=dev), 0
    for n, new in zip(lens, news):
        dead[base:base + max(0, new - n)] = True
        base += new
    for i, axis in enumerate(st["pair_axes"].tolist()):
        at = st["positions"][axis].long()
        c, s = st["cos"][at, i].to(f64)[:, None], st["sin"][at, i].to(f64)[:, None]
        lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        for x in (q, k):
            a, b = x[..., lo].clone(), x[..., hi].clone()
            x[..., lo], x[..., hi] = a * c - b * s, a * s + b * c

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


def _exact_logits(case, st):
    x = st["logits"].to(torch.float64)
    M, V = x.shape
    tokens = torch.full((M,), -1, dtype=torch.int64, device=x.device)
    bit = torch.arange(32, device=x.device)
    for m in range(M):
        row = x[m]
        if st["ids"] is not None:
            n, p = int(st["lengths"][m]), int(st["prompt"][m])
            seen = torch.unique(st["ids"][m, :n].long())
            old = row[seen]
            rep = float(st["repetition"][m])
            row[seen] = torch.where(old > 0, old / rep, old * rep)
            new, times = torch.unique(st["ids"][m, p:n].long(), return_counts=True)
            row[new] -= float(st["frequency"][m]) * times + float(st["presence"][m])
        if st["bias_ids"] is not None:
            last = {}
            for i, v in zip(st["bias_ids"][m].tolist(), st["bias"][m].tolist()):
                last[i] = v
            last.pop(-1, None)
            if last:
                row[list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device=x.device)
        ok = torch.ones(V, dtype=torch.bool, device=x.device)
        if st["allowed"] is not None:
            ok = ((st["allowed"][m][:, None] >> bit) & 1).bool().flatten()[:V]
            row[~ok] = -math.inf
        left = ok.nonzero()[:, 0]
        if len(left):
            best = row[left]
            tokens[m] = left[(best == best.max()).nonzero()[0, 0]]
    return {"logits": x, "tokens": tokens}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, st)
    return {"index": _exact_index, "sparse": _exact_sparse, "append": _exact_append}[case["op"]](case, st, *_lengths(case))
