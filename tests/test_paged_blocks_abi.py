"""Host side of the block index, the choice of blocks, attention over lists and
append by axes: what is refused before any CUDA call (these run without a GPU),
and the oracle's own cases."""
import ctypes

import numpy as np
import pytest

from oracle import blocks as B
from spectra_b200 import _lib as L
from spectra_b200 import paged as PG
from tests.test_paged_abi import COMMON, P, batch, cache


def at(x):
    return ctypes.addressof(x) if x is not None else None


def index(**kw):
    d = dict(codes=P, scales=P, block_size=32)
    d.update(kw)
    return L.BlockIndex(*d.values())


def update(c, b, i):
    return L.lib().spectra_paged_index_update(at(c), at(b), at(i), None)


def select(c, b, i, **kw):
    d = dict(dtype=L.DT_BF16, q_heads=4, q=P, q_ts=256, q_hs=64, count=8, first=1, last=1, blocks=P, b_ts=16, b_hs=8, stream=None)
    d.update(kw)
    return L.lib().spectra_paged_select_blocks(at(c), at(b), at(i), *d.values())


def attend(c, b, **kw):
    d = dict(dtype=L.DT_BF16, q_heads=4, q=P, q_ts=256, q_hs=64, out=P, o_ts=256, o_hs=64, scale=0.125, softcap=0.0,
             slopes=None, causal=1, window=0, blocks=P, b_ts=16, b_hs=8, count=8, block_size=32, ws=P, ws_bytes=1 << 30, stream=None)
    d.update(kw)
    return L.lib().spectra_paged_attention_blocks(at(c), at(b), *d.values())


def append(c, b, **kw):
    d = dict(dtype=L.DT_BF16, q_heads=4, q=P, q_ts=256, q_hs=64, q_out=P, qo_ts=256, qo_hs=64, k=P, k_ts=128, k_hs=64, v=P,
             v_ts=128, v_hs=64, cos=P, sin=P, cs_rows=256, cs_rs=32, rotary=64, interleaved=0, positions=P, pos_rs=3, axes=3,
             pair_axes=(0, 1, 2) * 11, stream=None)
    d.update(kw)
    if d["pair_axes"] is not None:
        held = (ctypes.c_uint8 * len(d["pair_axes"]))(*d["pair_axes"])
        d["pair_axes"] = ctypes.addressof(held)
    return L.lib().spectra_paged_kv_append_axes(at(c), at(b), *d.values())


@pytest.mark.parametrize("ckw,bkw,code", COMMON)
def test_every_entry_point_refuses_a_bad_cache_or_batch(ckw, bkw, code):
    c, b = cache(**ckw), batch(**bkw)
    assert update(c, b, index()) == code
    assert select(c, b, index()) == code
    assert attend(c, b) == code
    assert append(c, b) == code


@pytest.mark.parametrize("kw,code", [
    (dict(codes=None), L.ERR_NULL_POINTER),
    (dict(scales=None), L.ERR_NULL_POINTER),
    (dict(codes=P + 8), L.ERR_ALIGNMENT),
    (dict(scales=P + 2), L.ERR_ALIGNMENT),
    (dict(block_size=16), L.ERR_UNSUPPORTED),
    (dict(block_size=48), L.ERR_UNSUPPORTED),
    (dict(block_size=128), L.ERR_UNSUPPORTED),  # more than a page
    (dict(block_size=0), L.ERR_UNSUPPORTED),
    (dict(block_size=-64), L.ERR_UNSUPPORTED),
])
def test_a_bad_index_is_refused(kw, code):
    assert update(cache(), batch(), index(**kw)) == code
    assert select(cache(), batch(), index(**kw)) == code


def test_no_index_and_no_tokens():
    empty = batch(total=0)
    assert update(cache(), batch(), None) == L.ERR_NULL_POINTER and select(cache(), batch(), None) == L.ERR_NULL_POINTER
    assert update(cache(), empty, index()) == L.OK and select(cache(), empty, index()) == L.OK
    assert attend(cache(), empty) == L.OK and append(cache(), empty) == L.OK


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=L.DT_F32), L.ERR_DTYPE),
    (dict(q_heads=5), L.ERR_SHAPE),
    (dict(q_heads=0), L.ERR_SHAPE),
    (dict(count=0), L.ERR_SHAPE),
    (dict(count=L.MAX_LISTED_BLOCKS + 1), L.ERR_SHAPE),
    (dict(first=-1), L.ERR_SHAPE),
    (dict(last=0), L.ERR_SHAPE),
    (dict(first=5, last=4), L.ERR_SHAPE),
    (dict(first=2**62, last=2**62), L.ERR_SHAPE),
    (dict(q=None), L.ERR_NULL_POINTER),
    (dict(blocks=None), L.ERR_NULL_POINTER),
    (dict(q_ts=-1), L.ERR_STRIDE),
    (dict(b_ts=7), L.ERR_STRIDE),
    (dict(b_hs=7), L.ERR_STRIDE),
    (dict(q=P + 1), L.ERR_ALIGNMENT),
    (dict(blocks=P + 2), L.ERR_ALIGNMENT),
])
def test_the_choice_refuses(kw, code):
    assert select(cache(), batch(), index(), **kw) == code


def test_the_choice_refuses_more_blocks_than_it_ranks():
    wide = batch(width=1 << 21, table_stride=1 << 21, max_len=2**31 - 1)
    assert select(cache(), wide, index()) == L.ERR_SHAPE


@pytest.mark.parametrize("kw,code", [
    (dict(blocks=None), L.ERR_NULL_POINTER),
    (dict(blocks=P + 1), L.ERR_ALIGNMENT),
    (dict(b_ts=-1), L.ERR_STRIDE),
    (dict(b_hs=-1), L.ERR_STRIDE),
    (dict(count=0), L.ERR_SHAPE),
    (dict(count=L.MAX_LISTED_BLOCKS + 1), L.ERR_SHAPE),
    (dict(block_size=16), L.ERR_UNSUPPORTED),
    (dict(block_size=96), L.ERR_UNSUPPORTED),
    (dict(block_size=1 << 17), L.ERR_UNSUPPORTED),
    (dict(ws_bytes=4096), L.ERR_WORKSPACE),
    (dict(window=-1), L.ERR_SHAPE),
    (dict(scale=0.0), L.ERR_UNSUPPORTED),
])
def test_attention_over_lists_refuses(kw, code):
    assert attend(cache(), batch(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(positions=None), L.ERR_NULL_POINTER),
    (dict(pair_axes=None), L.ERR_NULL_POINTER),
    (dict(positions=P + 2), L.ERR_ALIGNMENT),
    (dict(axes=0), L.ERR_SHAPE),
    (dict(axes=5), L.ERR_SHAPE),
    (dict(axes=2), L.ERR_SHAPE),             # a pair on axis 2
    (dict(rotary=0), L.ERR_SHAPE),
    (dict(cs_rows=0), L.ERR_SHAPE),
    (dict(pos_rs=-3), L.ERR_STRIDE),
    (dict(cos=None), L.ERR_NULL_POINTER),
])
def test_append_by_axes_refuses(kw, code):
    assert append(cache(), batch(), **kw) == code


@pytest.mark.parametrize("call,err", [
    (lambda: PG.RotaryAxes([]), ValueError),
    (lambda: PG.RotaryAxes([0, 4]), ValueError),
    (lambda: PG.RotaryAxes([-1, 0]), ValueError),
    (lambda: PG.RotaryAxes.sections(3, -1), ValueError),
    (lambda: PG._block_size(16, 64), ValueError),
    (lambda: PG._block_size(128, 64), ValueError),
    (lambda: PG._block_size(96, 256), ValueError),
])
def test_python_refuses(call, err):
    with pytest.raises(err):
        call()


def test_sections():
    axes = PG.RotaryAxes.sections(2, 0, 3)
    assert axes.pair_axes == (0, 0, 2, 2, 2) and axes.axes == 3 and bytes(axes._c) == bytes([0, 0, 2, 2, 2])


def test_oracle_steps_bounds_and_lists():
    for most, want in ((0, 1), (127, 1), (127.5, 2), (64, 1), (63.5, 0.5), (63.75, 1), (254, 2), (1e-45, 2.0**-126), (3e38, 2.0**121)):
        assert B.step(most) == want and (most == 0 or most <= 127 * want)
    codes, s = B.bounds(np.array([[1.0, -3.0], [0.25, -2.9]]))
    assert s == 2.0**-5 and codes.tolist() == [[32, -92], [8, -96]]
    keys = np.random.default_rng(0).normal(size=(40, 16))
    codes, s = B.bounds(keys)
    q = np.random.default_rng(1).normal(size=(3, 16))
    c = B.query_codes(q)
    assert (B.scores(q, codes[None], np.array([s]))[0] >= (c @ keys.T).max() - 1e-9)  # a bound from above
    see = B.listed([2, 2, -1, 1, 3, 9], 30, 8)
    assert see.nonzero()[0].tolist() == list(range(16, 30))
    assert B.select(q, np.stack([codes] * 5), np.full(5, s), np.array([1, 1, 0, 1, 1], bool), 5, 3, 1, 1) == [0, 1, 4]


