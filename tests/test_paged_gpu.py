"""The paged INT4 KV cache (csrc/paged_kv.cu, paged_attn.cu, paged_prompt.cu)
against the oracle (oracle/paged.py): appended bytes and rotated queries bit
for bit, attention within a bound derived from its roundings."""
import numpy as np
import pytest
import torch

from oracle import paged as R
from spectra_b200 import kernels as SK
from spectra_b200 import paged as PG

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
TDT = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DIMS = list(PG.HEAD_DIMS)


def draw(shape, seed, dt, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * (1 + spread * (torch.rand(shape[-2:], generator=g) > 0.95))
    return x.to(TDT[dt])


def f32(t):
    return t.detach().cpu().float().numpy()


def angles(rotary, rows):
    if not rotary:
        return np.zeros((rows, 0), np.float32), np.zeros((rows, 0), np.float32)
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class Step:
    """A pool with sequences of the given lengths and a batch of their last `news` tokens."""

    def __init__(self, lens, news, heads, kv_heads, dim, page, dt, seed=0, spare=2, max_len=None, uniform=None):
        self.lens, self.news, self.heads, self.kv_heads, self.dim, self.dt = lens, news, heads, kv_heads, dim, dt
        self.page, self.seed = page, seed
        rng = np.random.default_rng(seed)
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + spare
        perm = rng.permutation(pages)
        self.tables = np.full((len(lens), max(counts + [1])), -1, np.int32)
        at = 0
        for b, c in enumerate(counts):
            self.tables[b, :c] = perm[at:at + c]
            at += c
        self.ref = R.Pool(pages, kv_heads, dim, page)
        self.total = sum(news)
        uniform = len(set(news)) == 1 if uniform is None else uniform
        cu = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=DEV)
        self.t_tables = torch.from_numpy(self.tables).to(DEV)
        self.t_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.batch = PG.TokenBatch(self.t_tables, self.t_lens, cu_q=None if uniform else cu,
                                   q_len=news[0] if uniform else None, total=self.total, max_q=max(news), max_len=max_len)
        self.first = np.concatenate([[0], np.cumsum(news)])

    def positions(self, b):
        return np.arange(self.lens[b] - self.news[b], self.lens[b])

    def fill(self, spread=3.0):
        """Every sequence's tokens into the reference pool, and the pool's bytes to the device."""
        for b, n in enumerate(self.lens):
            if n:
                k = f32(draw((n, self.kv_heads, self.dim), 1000 * self.seed + 2 * b, self.dt, spread))
                v = f32(draw((n, self.kv_heads, self.dim), 1000 * self.seed + 2 * b + 1, self.dt))
                self.ref.append(self.tables[b], np.arange(n), k, v)
        return self.upload()

    def upload(self):
        self.cache = PG.PagedKVCache.from_pool(torch.from_numpy(self.ref.to_bytes()).to(DEV), self.dim)
        return self.cache

    def check(self, q, out, **kw):
        """|out - exact| <= weights' and values' roundings * sum p |v| + the output's rounding."""
        dt = out.dtype
        qd, od = q.detach().cpu().double().numpy(), out.detach().cpu().double().numpy()
        scale = kw.pop("scale", self.dim ** -0.5)
        limit = kw.pop("limit", None)
        for b, n in enumerate(self.lens):
            rows = slice(self.first[b], self.first[b + 1])
            n = max(0, n if limit is None else min(n, limit))
            kv, held, steps = self.ref.values(self.tables[b], n)
            want, spread, size = R.attention(qd[rows], kv[0], kv[1], held, steps, self.positions(b), scale, **kw)
            # error of a score: keys or products rounded to 11 bits at most; fp32 sums of at most 1039 times a
            # group's queries, a few roundings each (2^-20); the cap's tanh; the bias and the scaling by log2 e
            eps = scale * (2.0**-11 * size[0] + 2.0**-20 * 1039 * size[1]) + 2.0**-21 * kw.get("softcap", 0.0)
            top = scale * size[0] + (np.max(kw["slopes"]) * n if kw.get("slopes") is not None else 0.0)
            eps = eps + 2.0**-21 * (top + 8)
            # of the result: weights and their sum, each off by e^eps and fp16's rounding; values' rounding
            rel = 2 * np.expm1(eps)[..., None] + 2 * 2.0**-11 + 2.0**-18
            tol = rel * spread + UNIT[dt] * np.abs(want) + 2.0**-24
            with np.errstate(invalid="ignore"):
                bad = ~(np.abs(od[rows] - want) <= tol)
            bad &= ~(np.isnan(od[rows]) & np.isnan(want))
            assert not bad.any(), (f"sequence {b}: {bad.sum()} of {bad.size} outside, worst "
                                   f"{np.nanmax(np.abs(od[rows] - want) / tol):.2f} of the bound")


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------

def append_and_check(st, q, k, v, rotary, interleaved, pool=None, ref_q=None, ref_k=None, ref_v=None):
    rows = max(max(st.lens), 1)
    cos, sin = angles(rotary, max(rows, st.batch._limit(pool or st.cache)))
    cache = pool or st.cache
    tc, ts = (torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV)) if rotary else (None, None)
    got = PG.paged_kv_append(cache, st.batch, k, v, q=q, cos=tc, sin=ts, interleaved=interleaved)
    for b in range(len(st.lens)):
        pos = st.positions(b)
        rows = slice(st.first[b], st.first[b + 1])
        real = pos >= 0
        at = np.maximum(pos, 0)
        kr = R.rotate(f32(k)[rows], cos[at], sin[at], interleaved)
        st.ref.append(st.tables[b], pos[real], kr[real], f32(v)[rows][real])
        if q is not None:
            turned = R.rotate(f32(q)[rows], cos[at], sin[at], interleaved)
            want = torch.from_numpy(np.where(real[:, None, None], turned, np.float32(0))).to(q.dtype)
            have = got[rows].cpu()
            assert torch.equal(have.view(torch.int16)[~have.isnan()], want.view(torch.int16)[~want.isnan()])
            assert torch.equal(have.isnan(), want.isnan())
    want = st.ref.to_bytes()
    have = cache.pool.cpu().numpy()
    assert np.array_equal(have, want), f"{(have != want).sum()} bytes of the pool differ"
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        ks, vs = PG.paged_kv_read(cache, st.batch, dtype=dt)
        for b in range(len(st.lens)):
            pos = st.positions(b)
            kv, _, _ = st.ref.values(st.tables[b], max(st.lens[b], 0))
            for t, w in ((ks, kv[0]), (vs, kv[1])):
                e = np.zeros((len(pos), st.kv_heads, st.dim))
                e[pos >= 0] = w[pos[pos >= 0]]
                e = torch.from_numpy(e).float().to(dt)
                h = t[st.first[b]:st.first[b + 1]].cpu()
                assert torch.equal(h.nan_to_num(7.0), e.nan_to_num(7.0))
    return got


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dt,interleaved,part", [("bf16", False, 1), ("f16", True, 1), ("bf16", True, 2), ("f16", False, 0)])
def test_append_bytes_and_read_back(dim, dt, interleaved, part):
    rotary = 0 if part == 0 else dim // part // 16 * 16
    st = Step([37, 1, 16, 81], [5, 1, 16, 33], 6, 2, dim, 16, dt, seed=dim + part)
    st.upload()
    q, k, v = (draw((st.total, h, dim), 5 + i, dt).to(DEV) for i, h in enumerate((6, 2, 2)))
    append_and_check(st, q, k, v, rotary, interleaved)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("lens", [[1], [16], [17, 33, 0, 300], [0, 0]])
def test_append_one_token_each(page, lens):
    st = Step(lens, [1] * len(lens), 8, 4, 64, page, "bf16", seed=3)
    st.upload()
    q, k, v = (draw((st.total, h, 64), 15 + i, "bf16").to(DEV) for i, h in enumerate((8, 4, 4)))
    got = append_and_check(st, q, k, v, 64, False)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()


def test_append_views_of_a_fused_projection_and_unaligned_rows():
    for off in (0, 1, 8):
        st = Step([40, 21], [40, 20], 4, 2, 64, 32, "bf16", seed=4)
        st.upload()
        wide = draw((st.total, 8 * 64 + 24), 9, "bf16").to(DEV)[:, off:off + 8 * 64].unflatten(1, (8, 64))
        append_and_check(st, wide[:, :4], wide[:, 4:6], wide[:, 6:], 64, False)
    st = Step([9], [9], 4, 2, 64, 32, "f16", seed=4)  # head-major tensors, and one shared by all tokens
    st.upload()
    q, k = (draw((h, 9, 64), 11, "f16").to(DEV).transpose(0, 1) for h in (4, 2))
    v = draw((1, 2, 64), 12, "f16").to(DEV).expand(9, 2, 64)
    append_and_check(st, q, k, v, 64, False)


def test_append_without_queries_and_into_a_given_tensor():
    st = Step([30], [30], 4, 2, 32, 16, "bf16")
    st.upload()
    k, v = (draw((30, 2, 32), 1 + i, "bf16").to(DEV) for i in range(2))
    assert append_and_check(st, None, k, v, 32, False) is None
    q = draw((30, 4, 32), 3, "bf16").to(DEV)
    cos, sin = (torch.from_numpy(a).to(DEV) for a in angles(32, 32))
    buf = torch.zeros(30, 6, 32, dtype=torch.bfloat16, device=DEV)
    out = PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=cos, sin=sin, out=buf[:, 1:5])
    assert out.data_ptr() == buf[:, 1:5].data_ptr()
    assert torch.equal(out, PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=cos, sin=sin))
    assert not buf[:, 0].any() and not buf[:, 5].any()


def test_append_groups_without_codes_constant_and_extreme():
    st = Step([20], [20], 2, 1, 64, 16, "bf16")
    st.upload()
    k, v = draw((20, 1, 64), 1, "bf16"), draw((20, 1, 64), 2, "bf16")
    k[0, 0, 3] = float("nan")
    k[1, 0, 40] = float("inf")
    v[2, 0, 5] = float("-inf")
    v[3, 0, 63] = float("nan")
    k[4, 0, :32] = 1e30
    v[5, 0, 0], v[5, 0, 1] = 40000.0, -40000.0  # spans more than its codes times the scale may
    k[6] = 0
    v[7] = 3.0       # one sign, constant
    k[8] = -2.5
    v[9] = 1e-9      # below the smallest scale
    k[10] = torch.linspace(0, 3e-6, 64).to(torch.bfloat16)  # subnormal scale
    v[11, 0, :32] = 60000.0
    v[12, 0, 5], v[13, 0, 5] = 65280.0, 65536.0  # the largest span below the bound, and the next
    append_and_check(st, draw((20, 2, 64), 3, "bf16").to(DEV), k.to(DEV), v.to(DEV), 0, False)
    ks, vs = PG.paged_kv_read(st.cache, st.batch, dtype=torch.float32)
    assert torch.isfinite(vs).all()
    nan = torch.zeros(20, 1, 64, dtype=torch.bool)
    for t, g in ((0, 0), (1, 1), (2, 0), (3, 1), (4, 0), (5, 0), (13, 0)):
        nan[t, 0, 32 * g:32 * g + 32] = True
    assert torch.equal(ks.isnan().cpu(), nan)
    # a group of one sign keeps half a step
    assert (vs[7] - 3.0).abs().max() <= 3.0 / 15 / 2 * 1.001 and (ks[8] + 2.5).abs().max() <= 2.5 / 15 / 2 * 1.001


def test_append_skips_bad_pages_and_positions_past_the_bound():
    st = Step([64, 64], [64, 64], 2, 2, 32, 16, "f16", max_len=50)
    st.tables[0, 1], st.tables[1, 2] = 10**6, -7
    st.t_tables.copy_(torch.from_numpy(st.tables))
    st.upload()
    q, k, v = (draw((128, 2, 32), i, "f16").to(DEV) for i in range(3))
    cos, sin = (torch.from_numpy(a).to(DEV) for a in angles(32, 50))
    got = PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=cos, sin=sin)
    for b in range(2):
        pos = np.arange(50)
        rows = slice(64 * b, 64 * b + 50)
        st.ref.append(st.tables[b], pos, R.rotate(f32(k)[rows], *angles(32, 50), False), f32(v)[rows])
    assert np.array_equal(st.cache.pool.cpu().numpy(), st.ref.to_bytes())
    assert not got[50:64].any() and not got[114:].any() and got[:50].any()


def test_append_into_pages_apart_and_past_two_gigabytes():
    dim, page, heads = 128, 64, 8
    each = heads * (page // 16) * PG.tile_bytes(dim)
    pages = 2**31 // each + 40
    raw = torch.zeros(pages * (each + 64), dtype=torch.uint8, device=DEV)
    pool = raw.as_strided((pages, heads, page // 16, PG.tile_bytes(dim)),
                          (each + 64, (page // 16) * PG.tile_bytes(dim), PG.tile_bytes(dim), 1))
    cache = PG.PagedKVCache.from_pool(pool, dim)
    st = Step([130], [130], 8, heads, dim, page, "bf16", spare=0)
    st.t_tables.copy_(torch.tensor([[pages - 1, 3, pages - 20]], dtype=torch.int32))
    k, v, q = (draw((130, heads, dim), i, "bf16").to(DEV) for i in range(3))
    PG.paged_kv_append(cache, st.batch, k, v)
    st.ref.append(st.tables[0], np.arange(130), f32(k), f32(v))
    want = st.ref.to_bytes()[st.tables[0]]
    for i, p in enumerate((pages - 1, 3, pages - 20)):
        assert np.array_equal(pool[p].cpu().numpy(), want[i])
    assert int(raw.count_nonzero()) == np.count_nonzero(want)
    st.check(q, PG.paged_attention(q, cache, st.batch))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (11, 1)])
def test_attention_one_token(dim, dt, heads, kv_heads):
    st = Step([1, 15, 16, 17, 33, 0, 129, 500], [1] * 8, heads, kv_heads, dim, 16, dt, seed=dim)
    st.fill()
    q = draw((8, heads, dim), 77, dt).to(DEV)
    out = PG.paged_attention(q, st.cache, st.batch)
    assert not out[5].any()
    st.check(q, out)


MASKS = {"plain": {}, "full": dict(causal=False), "window": dict(window=19), "cap": dict(softcap=5.0),
         "bias": dict(alibi=True), "all": dict(window=40, softcap=20.0, alibi=True),
         "full-window": dict(causal=False, window=7)}


def run_masked(st, q, mask, **kw):
    kw = {**MASKS[mask], **kw}
    slopes = None
    if kw.pop("alibi", False):
        slopes = np.exp2(-8.0 * np.arange(1, st.heads + 1) / st.heads).astype(np.float32)
    out = PG.paged_attention(q, st.cache, st.batch, alibi_slopes=None if slopes is None else torch.from_numpy(slopes).to(DEV),
                             **kw)
    st.check(q, out, slopes=slopes, **kw)
    return out


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("dim,dt", [(64, "bf16"), (128, "f16"), (96, "bf16"), (256, "bf16")])
@pytest.mark.parametrize("news", [[1] * 5, [2, 5, 1, 3, 9], [7] * 5])
def test_attention_masks_and_a_few_tokens(mask, dim, dt, news):
    st = Step([40, 200, 3, 64, 95], news, 4, 2, dim, 32, dt, seed=len(mask))
    st.fill()  # (sequence 2 may hold fewer tokens than are new: the first ones are padding)
    q = draw((st.total, 4, dim), 78, dt).to(DEV)
    run_masked(st, q, mask)


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("dim,dt", [(64, "bf16"), (128, "bf16"), (128, "f16"), (32, "f16"), (96, "bf16"), (256, "f16")])
def test_attention_prompts(mask, dim, dt):
    st = Step([130, 257, 64, 300], [130, 100, 1, 65], 4, 2, dim, 64, dt, seed=7)
    st.fill()
    q = draw((st.total, 4, dim), 79, dt).to(DEV)
    run_masked(st, q, mask)


@pytest.mark.parametrize("n", [128, 129, 383, 1000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (5, 1, 64), (2, 2, 128), (12, 1, 64)])
def test_attention_one_prompt(n, heads, kv_heads, dim):
    st = Step([n], [n], heads, kv_heads, dim, 16, "bf16", seed=n)
    st.fill()
    q = draw((n, heads, dim), 80, "bf16").to(DEV)
    run_masked(st, q, "plain")


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 4), (256, 4, 4), (256, 8, 2)])
@pytest.mark.parametrize("mask", ["plain", "all"])
def test_attention_prompts_of_many_sequences(dim, heads, kv_heads, mask):
    """Enough (sequence, head) pairs that no keys are split; chunks that look back, odd lengths, long sequences
    beside single tokens."""
    lens = [200, 129, 65, 331, 97, 128, 193, 64, 250, 130, 77, 160, 140, 99, 201, 127, 180, 1, 300, 150]
    news = [n if i % 3 else max(1, n // 2) for i, n in enumerate(lens)]
    news[5], news[8] = 1, 3
    st = Step(lens, news, heads, kv_heads, dim, 32, "bf16", seed=12)
    st.fill()
    q = draw((st.total, heads, dim), 91, "bf16").to(DEV)
    run_masked(st, q, mask)


def test_attention_wide_heads_prompt_and_repeatable_bits():
    st = Step([901], [700], 6, 2, 256, 64, "f16", seed=13)
    st.fill()
    q = draw((700, 6, 256), 92, "f16").to(DEV)
    out = run_masked(st, q, "cap")
    for _ in range(3):
        assert torch.equal(out, PG.paged_attention(q, st.cache, st.batch, softcap=5.0))


def test_attention_long_sequence_is_split_and_repeatable():
    st = Step([20011, 3, 7000], [1] * 3, 8, 2, 128, 64, "bf16", seed=1)
    st.fill()
    q = draw((3, 8, 128), 81, "bf16").to(DEV)
    out = PG.paged_attention(q, st.cache, st.batch)
    st.check(q, out)
    for _ in range(5):
        assert torch.equal(out, PG.paged_attention(q, st.cache, st.batch))


@pytest.mark.parametrize("news", [[1] * 3, [4, 2, 3], [150, 90, 200]])
def test_attention_sees_no_token_that_is_masked(news):
    """NaN keys and stale pages: only rows that see a poisoned token become NaN."""
    st = Step([150, 90, 200], news, 4, 2, 64, 16, "bf16", seed=5)
    st.fill()
    # a poisoned token in the middle of sequence 0, beyond the window of its last rows
    k, v = draw((1, 2, 64), 1, "bf16"), draw((1, 2, 64), 2, "bf16")
    v[0, 1, 40] = float("inf")
    st.ref.append(st.tables[0], [70], f32(k), f32(v))
    # what a page holds past the end of sequence 1 (90 tokens in pages of 16)
    page = st.tables[1, 5]
    st.ref.scales[page, :, 10:, 0] = np.nan
    st.ref.codes[page, :, 10:] = 15
    st.ref.scales[page, :, 10:, 1] = 4364.0  # the largest that is ever stored
    st.upload()
    q = draw((st.total, 4, 64), 82, "bf16").to(DEV)
    for mask in ("plain", "window", "full", "all"):
        out = run_masked(st, q, mask)
        assert torch.isfinite(out[st.first[1]:]).all()
    out = PG.paged_attention(q, st.cache, st.batch)
    pos = torch.from_numpy(st.positions(0))
    assert torch.equal(out[:st.first[1], 2:].isnan().all(-1).all(-1).cpu(), pos >= 70)
    assert torch.isfinite(out[:, :2]).all()  # the other key/value head


def test_attention_rows_of_infinite_and_nan_queries_stay_apart():
    for news in ([6, 2], [100, 40]):
        st = Step([100, 40], news, 4, 1, 64, 16, "f16", seed=6)
        st.fill()
        q = draw((st.total, 4, 64), 83, "f16")
        q[1, 2, 5] = float("nan")
        q[0, 1, 7] = float("inf")
        out = PG.paged_attention(q.to(DEV), st.cache, st.batch)
        bad = torch.zeros(st.total, 4, dtype=torch.bool)
        bad[1, 2] = True
        bad[0, 1] = out[0, 1].isnan().any().item()  # (inf: NaN unless every product is of one sign)
        assert torch.equal(out.isnan().any(-1).cpu(), bad)


def test_attention_bad_pages_are_not_seen():
    for news in ([1, 1], [80, 80]):
        st = Step([80, 80], news, 4, 2, 64, 16, "bf16", seed=8)
        st.fill()
        st.tables[0, 2], st.tables[1, 0], st.tables[1, 4] = -1, 10**8, 12345
        st.t_tables.copy_(torch.from_numpy(st.tables))
        q = draw((st.total, 4, 64), 84, "bf16").to(DEV)
        out = run_masked(st, q, "plain")
        st.tables[:] = -1  # no page at all: every row empty
        st.t_tables.fill_(-1)
        out = run_masked(st, q, "plain")
        assert not out.any()


def test_attention_lengths_past_the_bound_and_rows_past_the_batch():
    st = Step([100, 60], [1, 1], 4, 2, 64, 16, "bf16", max_len=70)
    st.fill()
    q = draw((2, 4, 64), 85, "bf16").to(DEV)
    st.check(q, PG.paged_attention(q, st.cache, st.batch), limit=70)
    # cu_q that ends before `total`: the rows after it belong to nobody
    cu = torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV)
    q = draw((9, 4, 64), 86, "bf16").to(DEV)
    batch = PG.TokenBatch(st.t_tables, st.t_lens, cu_q=cu, total=9, max_q=3)
    out = torch.full_like(q, 7.0)
    PG.paged_attention(q, st.cache, batch, out=out)
    assert not out[5:].any() and out[:5].any(-1).all()
    k, v = (draw((9, 2, 64), i, "bf16").to(DEV) for i in range(2))
    before = st.cache.pool.clone()
    turned = PG.paged_kv_append(st.cache, batch, k, v, q=q)
    assert not turned[5:].any() and torch.equal(turned[:5], q[:5])
    ks, _ = PG.paged_kv_read(st.cache, batch)
    assert not ks[5:].any()
    assert not torch.equal(before, st.cache.pool)


def test_attention_strided_queries_and_output():
    for news in ([3, 1], [70, 30]):
        for off in (0, 3, 8):
            st = Step([90, 30], news, 4, 2, 64, 16, "bf16", seed=9)
            st.fill()
            wide = draw((st.total, 6 * 64 + 16), 87, "bf16").to(DEV)
            q = wide[:, off:off + 4 * 64].unflatten(1, (4, 64))
            buf = torch.full((4, st.total, 66), 5.0, dtype=torch.bfloat16, device=DEV)
            out = PG.paged_attention(q, st.cache, st.batch, out=buf[..., 1:65].transpose(0, 1))
            st.check(q, out)
            assert (buf[..., 0] == 5.0).all() and (buf[..., 65] == 5.0).all()


def test_attention_scale_and_large_scores():
    for news in ([2, 2], [64, 64]):
        st = Step([100, 300], news, 4, 2, 64, 16, "bf16", seed=10)
        st.fill()
        q = (draw((st.total, 4, 64), 88, "bf16") * 16).to(DEV)  # sharp: one key takes nearly all
        run_masked(st, q, "plain", scale=0.5)
        run_masked(st, (q.float() * 2.0**-30).to(torch.bfloat16), "plain", scale=1e-3)  # flat
        tiny = st.cache.pool.clone()  # loud and quiet rows in one tile
        q[::3] *= 2.0**-20
        run_masked(st, q, "plain", scale=0.25)
        assert torch.equal(tiny, st.cache.pool)


def test_attention_on_another_stream_and_in_a_replayed_graph():
    st = Step([400, 77, 130], [1] * 3, 8, 2, 128, 32, "bf16", seed=11)
    st.fill()
    q = draw((3, 8, 128), 89, "bf16").to(DEV)
    want = PG.paged_attention(q, st.cache, st.batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = PG.paged_attention(q, st.cache, st.batch)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    k, v = (draw((3, 2, 128), 90 + i, "bf16").to(DEV) for i in range(2))
    cos, sin = (torch.from_numpy(a).to(DEV) for a in angles(128, 512))
    batch = PG.TokenBatch(st.t_tables, st.t_lens, max_len=448)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        PG.paged_attention(q, st.cache, batch)  # this stream's workspace
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        turned = PG.paged_kv_append(st.cache, batch, k, v, q=q, cos=cos, sin=sin)
        out = PG.paged_attention(turned, st.cache, batch)
    for lens in ([400, 77, 130], [401, 78, 0], [13, 2, 100]):
        st.lens = lens
        st.t_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(draw((3, 8, 128), 100 + lens[0], "bf16"))
        graph.replay()
        c, s = angles(128, 512)
        for b, n in enumerate(lens):
            if n:
                kr = R.rotate(f32(k)[b:b + 1], c[n - 1:n], s[n - 1:n], False)
                st.ref.append(st.tables[b], [n - 1], kr, f32(v)[b:b + 1])
        st.check(turned, out)


def test_no_wait_ran_out():
    torch.cuda.synchronize()
    assert SK.device_timeouts() == 0
