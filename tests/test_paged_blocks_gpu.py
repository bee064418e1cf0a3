"""Block index, choice of blocks and attention over lists of blocks
(csrc/paged_index.cu, paged_attn.cu) against the oracles: index and lists
exactly, attention within the bound of its roundings (tests/test_paged_gpu.py)."""
import numpy as np
import pytest
import torch

from oracle import blocks as B
from oracle import paged as R
from spectra_b200 import kernels as SK
from spectra_b200 import paged as PG
from tests.test_paged_gpu import DEV, UNIT, Step, draw, f32

pytestmark = pytest.mark.gpu


def want_index(st, block, lens=None):
    """Index of every full block of every sequence: codes and scales by page, as the oracle has them."""
    per = st.page // block
    pages, heads = st.ref.codes.shape[:2]
    codes = np.zeros((pages, heads, per, 2, st.dim), np.int8)
    scales = np.zeros((pages, heads, per), np.float32)
    for b, n in enumerate(lens or st.lens):
        keys = st.ref.values(st.tables[b], n)[0][0] if n else None
        for j in range(n // block):
            page = int(st.tables[b, j * block // st.page])
            if not 0 <= page < pages:
                continue
            for h in range(heads):
                at = (page, h, j % per)
                codes[at], scales[at] = B.bounds(keys[j * block:(j + 1) * block, h])
    return codes, scales


def same(index, want):
    codes, scales = want
    assert np.array_equal(index.codes.cpu().numpy(), codes)
    assert np.array_equal(index.scales.cpu().numpy(), scales)


def with_index(st, block):
    """The step's cache with an index of all its full blocks, from the oracle."""
    codes, scales = want_index(st, block)
    st.index_ref = codes, scales
    return PG.BlockIndex.from_buffers(st.cache, torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV))


def want_lists(st, q, block, count, first, last, limit=None):
    codes, scales = st.index_ref
    per, r = st.page // block, st.heads // st.kv_heads
    out = np.full((st.total, st.kv_heads, count), -1, np.int32)
    qd = q.detach().cpu().double().numpy()
    for b in range(len(st.lens)):
        for i, p in enumerate(st.positions(b)):
            if p < 0 or (limit is not None and p >= limit):
                continue
            t, n = st.first[b] + i, p // block + 1
            page = st.tables[b, np.arange(n) * block // st.page]
            held = (page >= 0) & (page < len(codes))
            at = np.where(held, page, 0)
            for h in range(st.kv_heads):
                j = np.arange(n) % per
                got = B.select(qd[t, h * r:(h + 1) * r], codes[at, h, j], scales[at, h, j], held, n, count, first, last)
                out[t, h, :len(got)] = got
    return out


# ---------------------------------------------------------------------------
# index
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dim", PG.HEAD_DIMS)
@pytest.mark.parametrize("page,block", [(32, 32), (128, 32), (64, 64), (256, 128)])
def test_index_of_prompts(dim, page, block):
    st = Step([1, 31, 32, 33, 0, 255, 256, 300], [1, 31, 32, 33, 0, 255, 256, 300], 4, 3, dim, page, "bf16", seed=dim)
    st.fill()
    index = PG.BlockIndex(st.cache, block)
    PG.paged_index_update(index, st.batch)
    same(index, want_index(st, block))


@pytest.mark.parametrize("news", [1, 3, 40])
def test_index_writes_the_blocks_that_the_new_tokens_filled_and_no_other(news):
    lens = [64, 63, 65, 128, 32, 31, 2, 0, 100]
    st = Step(lens, [news] * 9, 4, 2, 64, 64, "f16", seed=news)
    st.fill()
    index = PG.BlockIndex(st.cache, 32)
    index.codes.fill_(99)
    index.scales.fill_(-5.0)
    PG.paged_index_update(index, st.batch)
    codes, scales = want_index(st, 32)
    keep = np.ones(scales.shape, bool)
    for b, n in enumerate(lens):
        for j in range(max(0, n - news) // 32, n // 32):
            keep[st.tables[b, j // 2], :, j % 2] = False
    codes[keep], scales[keep] = 99, -5.0
    same(index, (codes, scales))


@pytest.mark.parametrize("dim,kv_heads,page,block", [(32, 16, 64, 32), (64, 16, 256, 256), (96, 12, 128, 64), (128, 16, 64, 64),
                                                      (256, 8, 128, 128), (128, 3, 512, 512)])
def test_index_of_more_sequences_than_are_laid_out_at_once(dim, kv_heads, page, block):
    lens = [block + (37 * i) % (3 * block) if i % 7 else 0 for i in range(150)]
    news = [max(1, n - (11 * i) % 40) for i, n in enumerate(lens)]
    st = Step(lens, news, kv_heads, kv_heads, dim, page, "bf16", seed=block)
    st.tables[9, 0] = -1
    st.t_tables.copy_(torch.from_numpy(st.tables))
    rng = np.random.default_rng(3)  # (codes drawn as they are: filling 150 sequences takes long)
    shape = st.ref.codes.shape
    st.ref.codes[:] = rng.integers(0, 16, shape, np.uint8)
    st.ref.scales[:] = rng.uniform(0.01, 3.0, st.ref.scales.shape).astype(np.float16)
    st.ref.zeros[:] = rng.integers(0, 16, st.ref.zeros.shape, np.uint8)
    st.upload()
    index = PG.BlockIndex(st.cache, block)
    PG.paged_index_update(index, st.batch)
    codes, scales = np.zeros(index.codes.shape, np.int8), np.zeros(index.scales.shape, np.float32)
    keys = ((st.ref.codes[:, :, :, 0].astype(np.float64).reshape(*shape[:3], -1, 32) - st.ref.zeros[:, :, :, 0, :, None])
            * st.ref.scales[:, :, :, 0, :, None].astype(np.float64)).reshape(*shape[:3], dim)
    for b, (n, new) in enumerate(zip(lens, news)):
        for j in range(max(0, n - new) // block, n // block):
            p, part = int(st.tables[b, j * block // page]), j % (page // block)
            for h in range(kv_heads if p >= 0 else 0):
                codes[p, h, part], scales[p, h, part] = B.bounds(keys[p, h, part * block:(part + 1) * block])
    same(index, (codes, scales))
    assert SK.device_timeouts() == 0


def test_index_of_keys_that_are_not_finite_constant_or_zero():
    st = Step([192], [192], 2, 2, 64, 64, "bf16")
    k, v = draw((192, 2, 64), 1, "bf16"), draw((192, 2, 64), 2, "bf16")
    k[5, 0, 40] = float("nan")
    k[70, 1, 3] = float("inf")
    k[128:160] = 0
    k[160:] = 3.0
    v[180, 1, 0] = float("nan")  # takes the key's group with it
    st.upload()
    PG.paged_kv_append(st.cache, st.batch, k.to(DEV), v.to(DEV))
    st.ref.append(st.tables[0], np.arange(192), f32(k), f32(v))
    index = PG.BlockIndex(st.cache, 32)
    PG.paged_index_update(index, st.batch)
    codes, scales = want_index(st, 32)
    same(index, (codes, scales))
    assert np.isinf(scales).sum() == 3 and (scales[st.tables[0, 2], :, 0] == 1).all()


def test_index_skips_bad_pages_and_positions_past_the_bound():
    st = Step([128, 128], [128, 128], 2, 2, 32, 32, "f16", max_len=70)
    st.tables[0, 1], st.tables[1, 0] = 10**6, -7
    st.t_tables.copy_(torch.from_numpy(st.tables))
    st.fill()
    index = PG.BlockIndex(st.cache, 32)
    PG.paged_index_update(index, st.batch)
    same(index, want_index(st, 32, [70, 70]))


def test_index_of_many_sequences_past_the_bound():
    # every third one's new tokens all lie past the bound, and what it counts must not move the others' blocks
    block, page, kv_heads, dim, limit = 32, 64, 16, 64, 96
    lens = [300 if i % 3 == 0 else 33 + 5 * i for i in range(40)]
    news = [40 if i % 3 == 0 else n for i, n in enumerate(lens)]
    st = Step(lens, news, kv_heads, kv_heads, dim, page, "bf16", max_len=limit)
    rng = np.random.default_rng(4)
    shape = st.ref.codes.shape
    st.ref.codes[:] = rng.integers(0, 16, shape, np.uint8)
    st.ref.scales[:] = rng.uniform(0.01, 3.0, st.ref.scales.shape).astype(np.float16)
    st.ref.zeros[:] = rng.integers(0, 16, st.ref.zeros.shape, np.uint8)
    st.upload()
    index = PG.BlockIndex(st.cache, block)
    PG.paged_index_update(index, st.batch)
    codes, scales = np.zeros(index.codes.shape, np.int8), np.zeros(index.scales.shape, np.float32)
    for b, (n, new) in enumerate(zip(lens, news)):
        keys = st.ref.values(st.tables[b], min(n, limit))[0][0]
        for j in range((n - new) // block, min(n, limit) // block):
            at = int(st.tables[b, j * block // page]), j % (page // block)
            for h in range(kv_heads):
                codes[at[0], h, at[1]], scales[at[0], h, at[1]] = B.bounds(keys[j * block:(j + 1) * block, h])
    assert scales.any()
    same(index, (codes, scales))
    assert SK.device_timeouts() == 0


def test_index_past_two_gigabytes_and_of_tokens_past_max_q():
    dim, page, heads = 128, 64, 8
    each = heads * (page // 16) * PG.tile_bytes(dim)
    pages = 2**31 // each + 40
    pool = torch.zeros(pages, heads, page // 16, PG.tile_bytes(dim), dtype=torch.uint8, device=DEV)
    cache = PG.PagedKVCache.from_pool(pool, dim)
    st = Step([130], [130], 8, heads, dim, page, "bf16", spare=0)
    st.t_tables.copy_(torch.tensor([[pages - 1, 3, pages - 20]], dtype=torch.int32))
    cu = torch.tensor([0, 130], dtype=torch.int32, device=DEV)
    batch = PG.TokenBatch(st.t_tables, st.t_lens, cu_q=cu, total=130, max_q=7)
    k, v = (draw((130, heads, dim), i, "bf16").to(DEV) for i in range(2))
    PG.paged_kv_append(cache, batch, k, v)
    st.ref.append(st.tables[0], np.arange(130), f32(k), f32(v))
    index = PG.BlockIndex(cache, 64)
    PG.paged_index_update(index, batch)
    codes, scales = want_index(st, 64)
    for i, p in enumerate((pages - 1, 3)):
        assert np.array_equal(index.codes[p].cpu().numpy(), codes[st.tables[0, i]])
        assert np.array_equal(index.scales[p].cpu().numpy(), scales[st.tables[0, i]])
    assert int(index.scales.count_nonzero()) == 2 * heads


# ---------------------------------------------------------------------------
# choice
# ---------------------------------------------------------------------------

def choose(st, q, block, count, first=1, last=1, limit=None, index=None):
    index = index or with_index(st, block)
    got = PG.paged_select_blocks(q, index, st.batch, count, first=first, last=last)
    want = want_lists(st, q, block, count, first, last, limit)
    assert got.dtype == torch.int32
    bad = (got.cpu().numpy() != want).any(-1)
    assert not bad.any(), f"{bad.sum()} of {bad.size} lists differ, first at {np.argwhere(bad)[0]}"
    return got


@pytest.mark.parametrize("dim", PG.HEAD_DIMS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (11, 1), (40, 1), (16, 2)])
def test_choice_one_token(dim, heads, kv_heads):
    st = Step([1, 32, 33, 900, 0, 2049, 31], [1] * 7, heads, kv_heads, dim, 64, "bf16", seed=dim)
    st.fill()
    choose(st, draw((7, heads, dim), 77, "bf16").to(DEV), 32, 6)


@pytest.mark.parametrize("count,first,last", [(1, 0, 1), (2, 1, 1), (5, 0, 5), (7, 3, 2), (64, 1, 1), (200, 0, 1)])
@pytest.mark.parametrize("news", [[1] * 4, [2, 5, 1, 9], [33, 64, 7, 100]])
def test_choice_counts_and_a_few_tokens(count, first, last, news):
    st = Step([3000, 700, 3, 2200], news, 4, 2, 64, 128, "f16", seed=count)
    st.fill()  # (sequence 2 may hold fewer tokens than are new: the first ones are padding)
    choose(st, draw((st.total, 4, 64), 78, "f16").to(DEV), 32, count, first, last)


@pytest.mark.parametrize("dim,heads,kv_heads,dt", [(128, 8, 2, "bf16"), (64, 16, 1, "f16"), (256, 4, 2, "bf16"), (96, 6, 2, "bf16"),
                                                   (32, 2, 2, "f16"), (128, 5, 1, "bf16")])
def test_choice_prompts(dim, heads, kv_heads, dt):
    st = Step([640, 257, 64, 1300], [640, 100, 1, 65], heads, kv_heads, dim, 64, dt, seed=7)
    st.fill()
    choose(st, draw((st.total, heads, dim), 79, dt).to(DEV), 32, 6, 1, 2)


def test_choice_with_equal_scores_takes_the_lowest():
    st = Step([32 * 40 + 5], [3], 4, 2, 64, 64, "bf16")
    one = draw((32, 2, 64), 1, "bf16")
    k = one.repeat(41, 1, 1)[:st.lens[0]]  # every block the same
    st.ref.append(st.tables[0], np.arange(st.lens[0]), f32(k), f32(k))
    st.upload()
    q = draw((3, 4, 64), 2, "bf16").to(DEV)
    got = choose(st, q, 32, 9, 2, 3)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 38, 39, 40]
    zero = choose(st, torch.zeros_like(q), 32, 9, 2, 3)  # (all scores 0)
    assert torch.equal(zero, got)


def test_choice_of_queries_of_any_size_and_not_finite():
    st = Step([2000, 1500], [8, 8], 4, 2, 128, 64, "bf16", seed=9)
    st.fill()
    q = draw((16, 4, 128), 3, "bf16")
    for i, f in enumerate((1e-38, 1e38, 3e-41, 1.0, 2.0**-126, 127.0)):
        q[i] = (q[i].float() / q[i].float().abs().amax() * f).to(torch.bfloat16)
    q[6, 1, 5], q[7, :, 3], q[8, 2, 0] = float("nan"), float("inf"), float("-inf")
    q[9] = 0
    choose(st, q.to(DEV), 64, 8)


def test_choice_puts_blocks_of_keys_that_are_not_finite_first_and_passes_over_bad_pages():
    st = Step([1000, 990], [2, 1], 4, 2, 64, 32, "bf16", seed=10)
    st.tables[0, 3], st.tables[0, 31], st.tables[1, 0] = 10**6, -7, -1
    st.t_tables.copy_(torch.from_numpy(st.tables))
    k, v = draw((1000, 2, 64), 1, "bf16"), draw((1000, 2, 64), 2, "bf16")
    k[300, 0, 7], k[640, 1, 9] = float("nan"), float("inf")
    for b, n in enumerate(st.lens):
        st.ref.append(st.tables[b], np.arange(n), f32(k)[:n], f32(v)[:n])
    st.upload()
    got = choose(st, draw((3, 4, 64), 5, "bf16").to(DEV), 32, 7, 2, 2)
    assert 300 // 32 in got[0, 0].tolist() and 640 // 32 in got[0, 1].tolist()
    assert not (got == 3)[:2].any() and not (got[:2] == 31).any() and not (got[2] == 0).any()


def test_choice_of_strided_queries_and_past_the_bound():
    st = Step([400, 300], [10, 7], 4, 2, 64, 64, "bf16", seed=11, max_len=396)
    st.fill()
    wide = draw((17, 8 * 64 + 24), 9, "bf16").to(DEV)
    for off in (0, 1, 8):
        q = wide[:, off:off + 8 * 64].unflatten(1, (8, 64))[:, 2:6]
        choose(st, q, 32, 5, limit=396)
    out = torch.empty(17, 2, 5, dtype=torch.int32, device=DEV)
    assert PG.paged_select_blocks(q, with_index(st, 32), st.batch, 5, out=out) is out


def test_choice_among_many_blocks():
    st = Step([32 * 9000 + 3], [1], 2, 1, 32, 4096, "bf16", seed=13)
    k = draw((st.lens[0], 1, 32), 1, "bf16")
    st.ref.append(st.tables[0], np.arange(st.lens[0]), f32(k), f32(k))
    st.upload()
    choose(st, draw((1, 2, 32), 4, "bf16").to(DEV), 32, 1024, 3, 4)
    choose(st, draw((1, 2, 32), 5, "bf16").to(DEV), 32, 33)


# ---------------------------------------------------------------------------
# attention over lists
# ---------------------------------------------------------------------------

def check_lists(st, q, out, blocks, block, slopes=None, limit=None, **kw):
    """As Step.check, row by row of the lists: the bound derived there."""
    dt, r = out.dtype, st.heads // st.kv_heads
    qd, od, lists = q.detach().cpu().double().numpy(), out.detach().cpu().double().numpy(), blocks.cpu().numpy()
    scale = st.dim ** -0.5
    for b, n in enumerate(st.lens):
        n = max(0, n if limit is None else min(n, limit))
        kv, held, steps = st.ref.values(st.tables[b], n)
        for i, p in enumerate(st.positions(b)):
            t = st.first[b] + i
            for h in range(st.kv_heads):
                hs = slice(h * r, (h + 1) * r)
                see = held & B.listed(lists[t, h], n, block)
                want, spread, size = R.attention(qd[t:t + 1, hs], kv[0][:, h:h + 1], kv[1][:, h:h + 1], see, steps[:, h:h + 1],
                                                 [p], scale, slopes=None if slopes is None else slopes[hs], **kw)
                eps = scale * (2.0**-11 * size[0] + 2.0**-20 * 1039 * size[1]) + 2.0**-21 * kw.get("softcap", 0.0)
                top = scale * size[0] + (np.max(slopes[hs]) * n if slopes is not None else 0.0)
                eps = eps + 2.0**-21 * (top + 8)
                rel = 2 * np.expm1(eps)[..., None] + 2 * 2.0**-11 + 2.0**-18
                tol = rel * spread + UNIT[dt] * np.abs(want) + 2.0**-24
                with np.errstate(invalid="ignore"):
                    bad = ~(np.abs(od[t:t + 1, hs] - want) <= tol)
                bad &= ~(np.isnan(od[t:t + 1, hs]) & np.isnan(want))
                assert not bad.any(), f"token {t}, head {h}: {bad.sum()} of {bad.size} outside"


def random_lists(st, count, block, seed, holes=True):
    """Ascending lists of random blocks, some with entries that are passed over."""
    rng = np.random.default_rng(seed)
    out = np.full((st.total, st.kv_heads, count), -1, np.int32)
    for b in range(len(st.lens)):
        for t in range(st.first[b], st.first[b + 1]):
            for h in range(st.kv_heads):
                n = max(1, -(-st.lens[b] // block)) + (2 if holes else 0)
                pick = np.sort(rng.choice(n, min(n, rng.integers(0, count + 1)), replace=False))
                at = np.sort(rng.choice(count, len(pick), replace=False)) if holes else np.arange(len(pick))
                out[t, h, at] = pick
    return torch.from_numpy(out).to(DEV)


CASES = {"plain": {}, "full": dict(causal=False), "window": dict(window=100), "cap": dict(softcap=5.0),
         "high cap": dict(softcap=300.0), "bias": dict(alibi=True), "all": dict(window=140, softcap=20.0, alibi=True)}


def attend(st, q, blocks, block, case="plain", limit=None, **kw):
    kw = {**CASES[case], **kw}
    slopes = None
    if kw.pop("alibi", False):
        slopes = np.exp2(-8.0 * np.arange(1, st.heads + 1) / st.heads).astype(np.float32)
    out = PG.paged_attention(q, st.cache, st.batch, blocks=blocks, block_size=block,
                             alibi_slopes=None if slopes is None else torch.from_numpy(slopes).to(DEV), **kw)
    check_lists(st, q, out, blocks, block, slopes, limit, **kw)
    return out


@pytest.mark.parametrize("dim", PG.HEAD_DIMS)
@pytest.mark.parametrize("dt,heads,kv_heads", [("bf16", 8, 2), ("f16", 3, 3), ("bf16", 11, 1), ("f16", 34, 2)])
def test_attention_over_lists_one_token(dim, dt, heads, kv_heads):
    st = Step([1, 31, 32, 33, 0, 500, 1000], [1] * 7, heads, kv_heads, dim, 32, dt, seed=dim)
    st.fill()
    q = draw((7, heads, dim), 77, dt).to(DEV)
    out = attend(st, q, random_lists(st, 9, 32, dim), 32)
    assert not out[4].any()


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("dim,dt", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("news", [[2, 5, 1, 3, 9], [7] * 5])
def test_attention_over_lists_masks_and_a_few_tokens(case, dim, dt, news):
    st = Step([140, 600, 3, 64, 295], news, 4, 2, dim, 32, dt, seed=len(case))
    st.fill()
    attend(st, draw((st.total, 4, dim), 78, dt).to(DEV), random_lists(st, 6, 64, 5), 64, case)


@pytest.mark.parametrize("page,block", [(16, 32), (16, 128), (64, 32), (64, 256), (1024, 64)])
def test_attention_over_lists_blocks_and_pages(page, block):
    """Blocks of several pages, pages of several blocks, pages that end inside a unit."""
    st = Step([777, 513, 90], [3, 1, 4], 4, 1, 64, page, "bf16", seed=page)
    st.fill()
    attend(st, draw((st.total, 4, 64), 79, "bf16").to(DEV), random_lists(st, 5, block, 6), block)


def test_attention_over_lists_passes_over_what_is_no_new_block():
    st = Step([640, 640], [2, 2], 4, 1, 64, 64, "bf16", seed=3)
    st.fill()
    q = draw((4, 4, 64), 80, "bf16").to(DEV)
    lists = torch.full((4, 1, 140), -1, dtype=torch.int32, device=DEV)
    lists[0, 0, :7] = torch.tensor([3, 3, 1, 5, 5, 4, 8])                 # 3, 5, 8
    lists[1, 0, 130:] = torch.tensor([0, 0, 9, 9, 10, 11, 2**31 - 1, -2**31, 6, 9])  # 0, 9
    lists[2, 0, 126:131] = torch.tensor([2, 7, 7, 2, 8])                  # 2, 7, 8: across a turn of 128
    out = attend(st, q, lists, 64)
    clean = torch.full((4, 1, 3), -1, dtype=torch.int32, device=DEV)
    clean[0, 0], clean[1, 0, :2], clean[2, 0] = torch.tensor([3, 5, 8]), torch.tensor([0, 9]), torch.tensor([2, 7, 8])
    assert not out[3].any()  # an empty list
    attend(st, q, clean, 64)


def test_attention_over_lists_of_every_block_is_the_whole_attention():
    st = Step([1200, 333, 64], [1, 4, 2], 8, 2, 128, 64, "bf16", seed=4)
    st.fill()
    q = draw((7, 8, 128), 81, "bf16").to(DEV)
    lists = torch.arange(19, dtype=torch.int32, device=DEV).expand(7, 2, 19)  # (one list for all: strides of 0)
    out = attend(st, q, lists, 64)
    st.check(q, out)


def test_attention_over_lists_bad_pages_bounds_and_rows_behind_the_last_sequence():
    st = Step([300, 200], [3, 2], 4, 2, 64, 32, "bf16", seed=5, max_len=290)
    st.tables[0, 2], st.tables[1, 4] = 10**6, -9
    st.t_tables.copy_(torch.from_numpy(st.tables))
    st.fill()
    q = draw((5, 4, 64), 82, "bf16").to(DEV)
    attend(st, q, random_lists(st, 8, 32, 7), 32, limit=290)
    cu = torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV)
    batch = PG.TokenBatch(st.t_tables, st.t_lens, cu_q=cu, total=9, max_q=2, max_len=290)
    q9 = draw((9, 4, 64), 83, "bf16").to(DEV)
    lists = torch.arange(8, dtype=torch.int32, device=DEV).expand(9, 2, 8).contiguous()
    out = torch.full_like(q9, 7.0)
    PG.paged_attention(q9, st.cache, batch, blocks=lists, block_size=32, out=out)
    assert not out[2].any() and not out[5:].any() and out[:2].any() and out[3:5].any()


def test_attention_over_long_lists_is_split_and_joined():
    st = Step([30000], [1], 4, 1, 64, 64, "bf16", seed=6)
    st.fill()
    q = draw((1, 4, 64), 84, "bf16").to(DEV)
    lists = torch.arange(0, 468, dtype=torch.int32, device=DEV)[None, None]
    a = attend(st, q, lists, 64)
    for _ in range(3):  # joined in one order whatever the CTAs' timing
        assert torch.equal(a, PG.paged_attention(q, st.cache, st.batch, blocks=lists, block_size=64))


@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 16, 1)])
def test_a_run_of_append_update_choose_attend(dim, heads, kv_heads):
    """Prompts, then single tokens, captured and replayed: index, lists and attention all along."""
    st = Step([0, 0, 0], [700, 330, 64], heads, kv_heads, dim, 64, "bf16", seed=21)
    st.tables = np.random.default_rng(1).permutation(36).reshape(3, 12).astype(np.int32)
    st.ref = R.Pool(36, kv_heads, dim, 64)
    st.upload()
    index = PG.BlockIndex(st.cache, 32)
    tables = torch.from_numpy(st.tables).to(DEV)
    lens = torch.tensor([700, 330, 64], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 700, 1030, 1094], dtype=torch.int32, device=DEV)
    prompt = PG.TokenBatch(tables, lens, cu_q=cu, total=1094, max_q=700)
    step = PG.TokenBatch(tables, lens)
    news = [700, 330, 64]

    def go(batch, q, k, v):
        PG.paged_kv_append(st.cache, batch, k, v)
        PG.paged_index_update(index, batch)
        blocks = PG.paged_select_blocks(q, index, batch, 6, first=1, last=2)
        return blocks, PG.paged_attention(q, st.cache, batch, blocks=blocks, block_size=32)

    def verify(q, k, v, blocks, out):
        st.lens = lens.tolist()
        st.news, st.first, st.total = news, np.concatenate([[0], np.cumsum(news)]), sum(news)
        for b in range(3):
            st.ref.append(st.tables[b], st.positions(b), f32(k)[st.first[b]:st.first[b + 1]], f32(v)[st.first[b]:st.first[b + 1]])
        st.index_ref = want_index(st, 32)
        same(index, st.index_ref)
        assert np.array_equal(blocks.cpu().numpy(), want_lists(st, q, 32, 6, 1, 2))
        check_lists(st, q, out, blocks, 32)

    draws = lambda n, seed: [draw((n, h, dim), seed + i, "bf16").to(DEV) for i, h in enumerate((heads, kv_heads, kv_heads))]  # noqa: E731
    qkv = draws(1094, 30)
    verify(*qkv, *go(prompt, *qkv))
    news = [1, 1, 1]
    held = draws(3, 40)
    lens.add_(1)
    verify(*held, *go(step, *held))  # (workspaces, kernel attributes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(1)
        res = go(step, *held)
    for i in range(40):
        for t, n in zip(held, draws(3, 50 + 3 * i)):
            t.copy_(n)
        graph.replay()
        if i % 13 == 0 or i > 35:
            verify(*held, *res)
        else:
            st.lens = lens.tolist()
            for b in range(3):
                st.ref.append(st.tables[b], [st.lens[b] - 1], f32(held[1])[b:b + 1], f32(held[2])[b:b + 1])
    assert SK.device_timeouts() == 0


def test_two_graphs_and_another_stream():
    st = Step([900, 800], [1, 1], 4, 2, 64, 64, "bf16", seed=22)
    st.fill()
    index = with_index(st, 32)
    q = draw((2, 4, 64), 85, "bf16").to(DEV)

    def go():
        blocks = PG.paged_select_blocks(q, index, st.batch, 5)
        return blocks, PG.paged_attention(q, st.cache, st.batch, blocks=blocks, block_size=32)

    want = go()
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = go()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = go()
        graphs.append((g, res))
    for g, _ in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    for res in [other] + [r for _, r in graphs]:
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
    check_lists(st, q, want[1], want[0], 32)
