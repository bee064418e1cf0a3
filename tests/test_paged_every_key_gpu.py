"""Attention over the paged INT4 cache, at bounds that a lost, doubled or
misplaced token would pass by far: marked values under equal weights, single
keys that take all the weight, and the root mean square error."""
import numpy as np
import pytest
import torch

from spectra_b200 import paged as PG
from tests.test_paged_caps_gpu import rms_check
from tests.test_paged_gpu import DEV, MASKS, Step, draw

pytestmark = pytest.mark.gpu


def marked(st, run):
    """Token t's value is 1 at feature (t // run + 7 head) % D of each head (exactly a code times its scale),
    0 elsewhere; keys as they come."""
    for b, n in enumerate(st.lens):
        if n:
            v = np.zeros((n, st.kv_heads, st.dim), np.float32)
            t, h = np.arange(n)[:, None], np.arange(st.kv_heads)
            v[t, h, (t // run + 7 * h) % st.dim] = 1.0
            k = draw((n, st.kv_heads, st.dim), 100 * st.seed + b, "f16").float().numpy()
            st.ref.append(st.tables[b], np.arange(n), k, v)
    return st.upload()


@pytest.mark.parametrize("run", [1, 16, 32, 64])
@pytest.mark.parametrize("dim,heads,kv_heads,lens,news", [
    (128, 8, 2, [20011, 3, 7000], [1, 1, 1]),          # split over many CTAs
    (64, 4, 1, [9001], [1]),
    (32, 12, 1, [3000, 517], [1, 1]),                  # two column tiles
    (256, 4, 2, [2999, 1031], [2, 5]),
    (64, 4, 2, [1000], [1000]),                        # a prompt, its keys split
    (128, 4, 4, [900, 300, 77], [400, 300, 1]),        # both kernels
    (256, 2, 1, [700], [300]),
])
def test_every_token_counts_once(run, dim, heads, kv_heads, lens, news):
    """Queries of 0: all weights are equal, and a feature of the result is how many of its tokens a row sees.
    One token more or less is 1 / (tokens of the feature), 1 / 160 at the least here (run 1 of the longest); the
    roundings are the weights' and the output's 2^-11 and the scale's of the value, also 2^-11 (its code is exact)."""
    st = Step(lens, news, heads, kv_heads, dim, 16, "f16", seed=61)
    marked(st, run)
    q = torch.zeros(st.total, heads, dim, dtype=torch.float16, device=DEV)
    for kw in ({}, dict(window=333), dict(causal=False)):
        out = PG.paged_attention(q, st.cache, st.batch, **kw).cpu().double().numpy()
        for b, n in enumerate(lens):
            rows = slice(st.first[b], st.first[b + 1])
            pos = st.positions(b)
            for i, p in enumerate(pos):
                lo = max(0, p - kw["window"] + 1) if "window" in kw else 0
                t = np.arange(lo, n if not kw.get("causal", True) else p + 1)
                for h in range(kv_heads):
                    count = np.bincount((t // run + 7 * h) % dim, minlength=dim)
                    have = out[rows][i, h * (heads // kv_heads):(h + 1) * (heads // kv_heads)] * len(t)
                    bad = np.abs(have - count) > count * 3 * 2.0**-11
                    assert not bad.any(), (b, p, h, np.abs(have - count).max())


@pytest.mark.parametrize("dim,heads,kv_heads,n,news", [
    (64, 64, 1, 2000, 1), (128, 32, 2, 6000, 1), (32, 16, 4, 700, 5), (256, 8, 1, 1500, 3),
    (64, 4, 1, 1500, 400), (128, 4, 2, 900, 300), (256, 2, 1, 800, 200), (96, 4, 2, 700, 350),
])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_a_key_that_takes_all_the_weight(dim, heads, kv_heads, n, news, dt):
    """Rows whose query is a multiple of one key: scores far above all others, so the result is that key's value,
    to the value's rounding (2^-11), the weight's (2^-11) and the output's."""
    st = Step([n], [news], heads, kv_heads, dim, 16, dt, seed=62)
    st.fill(spread=0.0)
    kv, _, _ = st.ref.values(st.tables[0], n)
    group, rng = heads // kv_heads, np.random.default_rng(3)
    pos = st.positions(0)
    for turn in range(4):
        # targets spread over all keys that a row sees, another set each turn
        target = (rng.permutation(n)[:news * heads] if news * heads <= n else rng.integers(0, n, news * heads)).reshape(news, heads)
        target = np.minimum(target, pos[:, None])
        h = np.arange(heads) // group
        q = torch.from_numpy(kv[0][target, h] * 16.0).to(torch.bfloat16 if dt == "bf16" else torch.float16).to(DEV)
        scores = np.einsum("ihd,nhd->ihn", q.cpu().double().numpy(), kv[0][:, h]) * dim ** -0.5
        scores[np.broadcast_to(np.arange(n) > pos[:, None, None], scores.shape)] = -np.inf
        top = np.take_along_axis(scores, target[..., None], -1)
        rest = scores.copy()
        np.put_along_axis(rest, target[..., None], -np.inf, -1)
        sure = top[..., 0] - rest.max(-1) > 25.0  # (with 2000 others at most: e^-25 * 2000 < 2^-25)
        assert sure.mean() > 0.5  # (of the inputs alone)
        want = kv[1][target, h]
        have = PG.paged_attention(q, st.cache, st.batch).cpu().double().numpy()
        unit = 2.0**-8 if dt == "bf16" else 2.0**-11
        tol = (unit + 2.0**-10) * np.abs(want) + 2.0**-18
        assert (np.abs(want) > tol)[sure].mean() > 0.8  # zeros would not do (a value's code may be 0)
        bad = np.abs(have - want)[sure] > tol[sure]
        assert not bad.any(), f"{bad.any(-1).sum()} of {len(bad)} rows"


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv_heads,lens,news", [
    (128, 8, 2, [20011, 3, 7000], [1, 1, 1]),
    (64, 16, 2, [3000, 100, 517, 1], [2, 5, 9, 1]),
    (256, 4, 2, [2500, 999], [1, 3]),
    (128, 4, 2, [700], [700]),
    (64, 4, 4, [600, 520, 77], [300, 200, 1]),
    (256, 4, 1, [500, 400], [180, 150]),
    (32, 4, 2, [400, 900], [300, 100]), (96, 4, 2, [400, 900], [300, 100]),
])
def test_root_mean_square_error(mask, dt, dim, heads, kv_heads, lens, news):
    """Scores of a few units; a lost unit of 32 of 20011 keys would move a result by 4 % of itself."""
    st = Step(lens, news, heads, kv_heads, dim, 32, dt, seed=63)
    st.fill(spread=0.0)
    q = draw((st.total, heads, dim), 64, dt, 0.0).to(DEV)
    kw = dict(MASKS[mask])
    slopes = None
    if kw.pop("alibi", False):
        slopes = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32)
    out = PG.paged_attention(q, st.cache, st.batch, alibi_slopes=None if slopes is None else torch.from_numpy(slopes).to(DEV), **kw)
    rms_check(st, q, out, slopes=slopes, **kw)
