"""Host side of the paged INT4 KV cache: what the C entry points and the Python
functions refuse before any CUDA call (so these run without a GPU), and the
oracle's layout and quantiser."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as R
from spectra_b200 import _lib as L
from spectra_b200 import paged as PG

P = 0x10000  # a fake device address: every call below fails its checks first


def cache(**kw):
    d = dict(pool=P, page_stride=2 * 4 * 1216, num_pages=8, kv_heads=2, head_dim=64, page_size=64)
    d.update(kw)
    return L.PagedCache(*d.values())


def batch(**kw):
    d = dict(block_tables=P, table_stride=4, width=4, seq_lens=P, cu_q=None, batch=3, q_len=1, total=3, max_q=1, max_len=256)
    d.update(kw)
    return L.TokenBatch(*d.values())


def append(c, b, **kw):
    d = dict(dtype=L.DT_BF16, q_heads=4, q=P, q_ts=256, q_hs=64, q_out=P, qo_ts=256, qo_hs=64, k=P, k_ts=128, k_hs=64, v=P,
             v_ts=128, v_hs=64, cos=P, sin=P, cs_rows=256, cs_rs=32, rotary=64, interleaved=0, stream=None)
    d.update(kw)
    return L.lib().spectra_paged_kv_append(ctypes.addressof(c) if c else None, ctypes.addressof(b) if b else None, *d.values())


def attend(c, b, **kw):
    d = dict(dtype=L.DT_BF16, q_heads=4, q=P, q_ts=256, q_hs=64, out=P, o_ts=256, o_hs=64, scale=0.125, softcap=0.0,
             slopes=None, causal=1, window=0, ws=P, ws_bytes=1 << 30, stream=None)
    d.update(kw)
    return L.lib().spectra_paged_attention(ctypes.addressof(c) if c else None, ctypes.addressof(b) if b else None, *d.values())


def read(c, b, k=P, v=P, dt=L.DT_F32):
    return L.lib().spectra_paged_kv_read(ctypes.addressof(c) if c else None, ctypes.addressof(b) if b else None, k, v, dt, None)


COMMON = [
    (dict(head_dim=80), {}, L.ERR_UNSUPPORTED),
    (dict(head_dim=0), {}, L.ERR_UNSUPPORTED),
    (dict(page_size=48), {}, L.ERR_UNSUPPORTED),
    (dict(page_size=8), {}, L.ERR_UNSUPPORTED),
    (dict(kv_heads=0), {}, L.ERR_SHAPE),
    (dict(num_pages=-1), {}, L.ERR_SHAPE),
    (dict(pool=None), {}, L.ERR_NULL_POINTER),
    (dict(pool=P + 8), {}, L.ERR_ALIGNMENT),
    (dict(page_stride=2 * 4 * 1216 + 8), {}, L.ERR_ALIGNMENT),
    (dict(page_stride=2 * 4 * 1216 - 16), {}, L.ERR_STRIDE),
    ({}, dict(block_tables=None), L.ERR_NULL_POINTER),
    ({}, dict(seq_lens=None), L.ERR_NULL_POINTER),
    ({}, dict(seq_lens=P + 2), L.ERR_ALIGNMENT),
    ({}, dict(cu_q=P + 1), L.ERR_ALIGNMENT),
    ({}, dict(table_stride=3), L.ERR_STRIDE),
    ({}, dict(batch=-1), L.ERR_SHAPE),
    ({}, dict(batch=0), L.ERR_SHAPE),
    ({}, dict(total=-1), L.ERR_SHAPE),
    ({}, dict(total=4), L.ERR_SHAPE),       # more rows than batch * q_len
    ({}, dict(q_len=0), L.ERR_SHAPE),
    ({}, dict(max_q=0), L.ERR_SHAPE),
    ({}, dict(max_len=-1), L.ERR_SHAPE),
    ({}, dict(total=1 << 40, cu_q=P), L.ERR_SHAPE),
]


@pytest.mark.parametrize("ckw,bkw,code", COMMON)
def test_every_entry_point_refuses_a_bad_cache_or_batch(ckw, bkw, code):
    c, b = cache(**ckw), batch(**bkw)
    assert append(c, b) == code
    assert attend(c, b) == code
    assert read(c, b) == code


def test_null_structures_and_empty_batches():
    c, b = cache(), batch()
    for f in (append, attend, read):
        assert f(None, b) == L.ERR_NULL_POINTER
        assert f(c, None) == L.ERR_NULL_POINTER
        assert f(c, batch(batch=0, total=0, q_len=1, max_q=0)) == L.OK  # nothing to do, nothing launched


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=L.DT_F32), L.ERR_DTYPE),
    (dict(rotary=72), L.ERR_SHAPE),
    (dict(rotary=24), L.ERR_SHAPE),
    (dict(rotary=-16), L.ERR_SHAPE),
    (dict(rotary=4, interleaved=1), L.ERR_SHAPE),
    (dict(cs_rows=255), L.ERR_SHAPE),
    (dict(cs_rs=31), L.ERR_SHAPE),
    (dict(q_heads=0), L.ERR_SHAPE),
    (dict(k=None), L.ERR_NULL_POINTER),
    (dict(v=None), L.ERR_NULL_POINTER),
    (dict(q_out=None), L.ERR_NULL_POINTER),
    (dict(cos=None), L.ERR_NULL_POINTER),
    (dict(sin=P + 2), L.ERR_ALIGNMENT),
    (dict(k=P + 1), L.ERR_ALIGNMENT),
    (dict(v_ts=-128), L.ERR_STRIDE),
])
def test_append_refuses(kw, code):
    assert append(cache(), batch(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=L.DT_F32), L.ERR_DTYPE),
    (dict(q_heads=3), L.ERR_SHAPE),
    (dict(q_heads=0), L.ERR_SHAPE),
    (dict(window=-1), L.ERR_SHAPE),
    (dict(scale=0.0), L.ERR_UNSUPPORTED),
    (dict(scale=float("nan")), L.ERR_UNSUPPORTED),
    (dict(scale=float("inf")), L.ERR_UNSUPPORTED),
    (dict(softcap=-1.0), L.ERR_UNSUPPORTED),
    (dict(softcap=float("nan")), L.ERR_UNSUPPORTED),
    (dict(q=None), L.ERR_NULL_POINTER),
    (dict(out=None), L.ERR_NULL_POINTER),
    (dict(ws=None), L.ERR_NULL_POINTER),
    (dict(ws=P + 8), L.ERR_ALIGNMENT),
    (dict(slopes=P + 2), L.ERR_ALIGNMENT),
    (dict(q_hs=-64), L.ERR_STRIDE),
    (dict(ws_bytes=1000), L.ERR_WORKSPACE),
])
def test_attention_refuses(kw, code):
    assert attend(cache(), batch(), **kw) == code


def test_attention_refuses_rows_that_32_bits_do_not_count():
    b = batch(cu_q=P, total=1 << 30, max_q=1 << 30)
    assert attend(cache(), b) == L.ERR_SHAPE
    assert attend(cache(kv_heads=1, page_stride=4 * 1216), b, q_heads=2) == L.ERR_SHAPE


def test_read_refuses():
    assert read(cache(), batch(), dt=L.DT_I32) == L.ERR_DTYPE
    assert read(cache(), batch(), k=None) == L.ERR_NULL_POINTER
    assert read(cache(), batch(), v=P + 8) == L.ERR_ALIGNMENT


def test_python_refuses_wrong_pools_and_batches():
    with pytest.raises(ValueError, match="head_dim"):
        PG.PagedKVCache(4, 2, 80)
    with pytest.raises(ValueError, match="page_size"):
        PG.PagedKVCache(4, 2, 64, page_size=40)
    with pytest.raises(RuntimeError, match="CUDA"):
        PG.PagedKVCache(4, 2, 64, device="cpu")
    pool = torch.zeros(4, 2, 4, 1216, dtype=torch.uint8)
    with pytest.raises(ValueError, match="pool must be"):
        PG.PagedKVCache.from_pool(pool, 128)
    with pytest.raises(TypeError, match="uint8"):
        PG.PagedKVCache.from_pool(pool.int(), 64)
    with pytest.raises(ValueError, match="contiguous"):
        PG.PagedKVCache.from_pool(pool.transpose(1, 2).contiguous().transpose(1, 2), 64)
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        PG.TokenBatch(t, n)
    with pytest.raises(TypeError, match="int32"):
        PG.TokenBatch(t.long(), n)


@pytest.mark.parametrize("dim", PG.HEAD_DIMS)
def test_oracle_layout_is_the_documented_one(dim):
    """Byte by byte from the header's description, for one tile."""
    G = dim // 32
    rng = np.random.default_rng(dim)
    pool = R.Pool(1, 1, dim, 16)
    pool.codes[:] = rng.integers(0, 16, pool.codes.shape)
    pool.scales[:] = rng.normal(size=pool.scales.shape)
    pool.zeros[:] = rng.integers(0, 16, pool.zeros.shape)
    b = pool.to_bytes().reshape(-1)
    assert b.size == PG.tile_bytes(dim)
    word = lambda at: int(b[at:at + 4].view(np.uint32)[0])  # noqa: E731
    for t in range(16):
        for g in range(G):
            for c in range(4):
                w = word(128 * G * (t // 8) + 4 * ((t % 8 * 4 + c) * G + g))
                assert [w >> 4 * i & 15 for i in range(8)] == list(pool.codes[0, 0, t, 0, 32 * g + 8 * c:][:8])
            for l in range(8):  # noqa: E741
                w = word(256 * G + 128 * G * (t // 8) + 4 * ((l * 4 + t % 8 // 2) * G + g)) >> 16 * (t % 2)
                assert [w >> 4 * i & 15 for i in range(4)] == list(pool.codes[0, 0, t, 1, 32 * g + 4 * l:][:4])
            half = lambda at: b[at:at + 2].view(np.float16)[0]  # noqa: E731
            assert half(512 * G + 2 * (t * G + g)) == pool.scales[0, 0, t, 0, g]
            assert half(544 * G + 2 * ((t // 2 * G + g) * 2 + t % 2)) == pool.scales[0, 0, t, 1, g]
            assert b[576 * G + t * G + g] == pool.zeros[0, 0, t, 0, g]
            assert b[592 * G + (t // 2 * G + g) * 2 + t % 2] == pool.zeros[0, 0, t, 1, g]


def test_oracle_quantiser_is_within_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(500, 2, 64)).astype(np.float32)
    x[100:200] += 5.0  # one sign
    x[200:300] *= 1e-3
    q, s, z = R.quantize(x, -x)
    for i, src in ((0, x), (1, -x)):
        g = src.reshape(500, 2, 2, 32)
        v = (q[..., i, :].reshape(g.shape).astype(np.float64) - z[..., i, :, None]) * s[..., i, :, None].astype(np.float64)
        # half a step, and half a step more where the zero point and the code both round up against the last code
        assert (np.abs(v - g) <= s[..., i, :, None].astype(np.float64) * (0.5 + 15 * 2.0**-11)).mean() > 0.99
        assert (np.abs(v - g) <= s[..., i, :, None].astype(np.float64) * (1.0 + 15 * 2.0**-11)).all()
