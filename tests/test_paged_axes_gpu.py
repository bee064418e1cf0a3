"""Append with positions of several axes (csrc/paged_kv.cu) against the oracle:
bytes of the pool and rotated queries bit for bit."""
import numpy as np
import pytest
import torch

from oracle import paged as R
from spectra_b200 import paged as PG
from tests.test_paged_gpu import DEV, Step, angles, draw, f32

pytestmark = pytest.mark.gpu


def rows_of(pos, pair_axes, cos, sin):
    """cos and sin [T, pairs] of positions [axes, T]; NaN where a position is outside the table."""
    at = np.asarray(pos)[np.asarray(pair_axes)].T.astype(np.int64)
    ok = (at >= 0) & (at < len(cos))
    i = np.arange(cos.shape[1])
    pick = lambda t: np.where(ok, t[np.where(ok, at, 0), i], np.float32(np.nan))  # noqa: E731
    return pick(cos), pick(sin)


def append(st, pair_axes, pos, table_rows, interleaved=False, heads=4, seed=1, dt="bf16", axes=None):
    q, k, v = (draw((st.total, h, st.dim), seed + i, dt).to(DEV) for i, h in enumerate((heads, st.kv_heads, st.kv_heads)))
    cos, sin = angles(2 * len(pair_axes), table_rows)
    st.upload()
    got = PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=torch.from_numpy(cos).to(DEV), sin=torch.from_numpy(sin).to(DEV),
                             interleaved=interleaved, positions=pos.to(DEV), axes=axes or PG.RotaryAxes(pair_axes))
    check(st, got, q, k, v, pos, pair_axes, cos, sin, interleaved)
    return got


def check(st, got, q, k, v, pos, pair_axes, cos, sin, interleaved):
    c, s = rows_of(pos.numpy() if pos.dim() == 2 else pos.numpy()[None], pair_axes, cos, sin)
    for b in range(len(st.lens)):
        at, rows = st.positions(b), slice(st.first[b], st.first[b + 1])
        real = at >= 0
        kr = R.rotate(f32(k)[rows], c[rows], s[rows], interleaved)
        st.ref.append(st.tables[b], at[real], kr[real], f32(v)[rows][real])
        turned = R.rotate(f32(q)[rows], c[rows], s[rows], interleaved)
        want = torch.from_numpy(np.where(real[:, None, None], turned, np.float32(0))).to(q.dtype)
        have = got[rows].cpu()
        assert torch.equal(have.isnan(), want.isnan())
        assert torch.equal(have.view(torch.int16)[~have.isnan()], want.view(torch.int16)[~want.isnan()])
    assert np.array_equal(st.cache.pool.cpu().numpy(), st.ref.to_bytes())


def random_positions(axes, total, rows, seed):
    return torch.randint(0, rows, (axes, total), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("dim", PG.HEAD_DIMS)
@pytest.mark.parametrize("order", ["sections", "turns", "random"])
@pytest.mark.parametrize("dt,interleaved,part", [("bf16", False, 1), ("f16", True, 1), ("bf16", True, 2), ("f16", False, 2)])
def test_three_axes(dim, order, dt, interleaved, part):
    half = dim // part // 16 * 16 // 2
    rng = np.random.default_rng(dim)
    pair_axes = {"sections": [0] * (half // 4) + [1] * (half // 4) + [2] * (half - half // 4 * 2),
                 "turns": [i % 3 for i in range(half)], "random": [2] + rng.integers(0, 3, half - 1).tolist()}[order]
    st = Step([37, 1, 16, 81], [5, 1, 16, 33], 4, 2, dim, 16, dt, seed=dim + part)
    append(st, pair_axes, random_positions(3, st.total, 500, dim), 500, interleaved, dt=dt)


@pytest.mark.parametrize("axes", [1, 2, 4])
def test_other_numbers_of_axes_and_single_tokens(axes):
    st = Step([17, 33, 0, 300], [1] * 4, 4, 2, 64, 64, "bf16", seed=3)
    append(st, [i % axes for i in range(32)], random_positions(axes, 4, 90, axes), 90)


def test_a_tokens_own_position_on_every_axis_is_the_plain_append():
    st = Step([50, 7], [50, 7], 4, 2, 128, 32, "bf16", seed=4)
    q, k, v = (draw((57, h, 128), i, "bf16").to(DEV) for i, h in enumerate((4, 2, 2)))
    cos, sin = (torch.from_numpy(a).to(DEV) for a in angles(128, 64))
    own = torch.cat([torch.arange(50), torch.arange(7)]).to(torch.int32).to(DEV)
    st.upload()
    a = PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=cos, sin=sin)
    pool = st.cache.pool.clone()
    for pos, axes in ((own.expand(3, 57), PG.RotaryAxes.sections(16, 24, 24)), (own, None), (own[None], None)):
        st.cache.pool.zero_()
        b = PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=cos, sin=sin, positions=pos, axes=axes)
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and torch.equal(pool, st.cache.pool)


def test_rows_outside_the_table_turn_into_nan_and_no_other():
    st = Step([40], [40], 4, 2, 64, 16, "bf16", seed=5)
    pos = random_positions(3, 40, 30, 5)
    pos[0, 3], pos[1, 9], pos[2, 11], pos[2, 12], pos[0, 39] = 30, -1, 2**31 - 1, -2**31, 29
    got = append(st, [0] * 8 + [1] * 12 + [2] * 12, pos, 30)
    assert got.isnan().any(-1).any(-1).nonzero()[:, 0].tolist() == [3, 9, 11, 12]


def test_the_table_may_be_shorter_than_the_cache_and_positions_strided():
    st = Step([600, 601], [1, 1], 4, 2, 64, 64, "f16", seed=6, max_len=1024)
    wide = torch.full((4, 10), 10**6, dtype=torch.int32)
    wide[:3, 4:6] = random_positions(3, 2, 20, 6)
    append(st, [i % 3 for i in range(32)], wide[:3, 4:6], 20, dt="f16")
    st = Step([600, 601], [1, 1], 4, 2, 64, 64, "f16", seed=6, max_len=1024)
    pos = random_positions(2, 6, 20, 7).t()[::2]  # tokens before axes: brought into order
    append(st, [0] * 16 + [1] * 16, pos[:2].clone().as_strided((2, 2), (1, 2)), 20, dt="f16")


def test_padding_bad_pages_and_a_captured_step():
    st = Step([3, 64, 20], [5, 30, 20], 4, 2, 64, 16, "bf16", seed=8)
    st.tables[1, 3] = 10**6
    st.t_tables.copy_(torch.from_numpy(st.tables))
    axes, pair = PG.RotaryAxes.sections(8, 12, 12), [0] * 8 + [1] * 12 + [2] * 12
    pos = random_positions(3, 55, 64, 9)
    append(st, pair, pos, 64, axes=axes)
    st = Step([9, 40], [1, 1], 4, 2, 64, 16, "bf16", seed=9)
    st.upload()
    q, k, v = (draw((2, h, 64), 20 + i, "bf16").to(DEV) for i, h in enumerate((4, 2, 2)))
    cos, sin = angles(64, 64)
    tc, ts, held = torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    call = lambda: PG.paged_kv_append(st.cache, st.batch, k, v, q=q, cos=tc, sin=ts, positions=held, axes=axes)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2):
        pos = random_positions(3, 2, 64, seed)
        held.copy_(pos)
        graph.replay()
        check(st, got, q, k, v, pos, pair, cos, sin, False)
