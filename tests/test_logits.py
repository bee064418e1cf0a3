"""Host side of the rules on logits: what the C entry point and the Python
functions refuse before any CUDA call, and the oracle's own cases."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import logits as R
from spectra_b200 import _lib as L
from spectra_b200 import logits as LG

MANY = dict(M=200, N=20000, x_rs=20000, out_rs=20000)  # two kernels, with a workspace
P = 0x10000  # a fake device address: every call below fails its checks first


def adjust(rules=None, **kw):
    r = dict(ids=P, ids_stride=8, max_ids=8, lengths=P, prompt_lengths=P, repetition=P, frequency=P, presence=P, bias_ids=P,
             bias_ids_stride=4, bias=P, bias_stride=4, n_bias=4, allowed=P, allowed_stride=4, allowed_words=4)
    r.update(rules or {})
    d = dict(x=P, x_dtype=L.DT_BF16, x_rs=100, M=2, N=100, offset=0, out=P, out_dtype=L.DT_BF16, out_rs=100, idx=P, val=P, ws=P, ws_bytes=1 << 20,
             stream=None)
    d.update(kw)
    c = L.LogitRules(*r.values())
    return L.lib().spectra_adjust_logits(ctypes.addressof(c) if rules != "null" else None, *d.values())


@pytest.mark.parametrize("rules,kw,code", [
    ({}, dict(x=None), L.ERR_NULL_POINTER),
    ({}, dict(out=None, idx=None, val=None), L.ERR_NULL_POINTER),
    ({}, dict(idx=None), L.ERR_NULL_POINTER),                 # a value without its token
    ({}, dict(N=0), L.ERR_SHAPE),
    ({}, dict(M=-1), L.ERR_SHAPE),
    ({}, dict(N=1 << 31, x_rs=1 << 31), L.ERR_SHAPE),
    ({}, dict(offset=-1), L.ERR_SHAPE),
    ({}, dict(offset=2**31 - 164), L.ERR_SHAPE),
    ({}, dict(offset=29), L.ERR_SHAPE),                       # 129 bits in 4 words
    (dict(allowed_words=3), {}, L.ERR_SHAPE),
    (dict(max_ids=L.MAX_RULE_IDS + 1), {}, L.ERR_SHAPE),
    (dict(max_ids=-1), {}, L.ERR_SHAPE),
    (dict(n_bias=L.MAX_RULE_BIASES + 1), {}, L.ERR_SHAPE),
    (dict(n_bias=-1), {}, L.ERR_SHAPE),
    ({}, dict(x_dtype=L.DT_I32), L.ERR_DTYPE),
    ({}, dict(out_dtype=L.DT_I64), L.ERR_DTYPE),
    ({}, dict(x_rs=99), L.ERR_STRIDE),
    ({}, dict(out_rs=99), L.ERR_STRIDE),
    (dict(ids_stride=-8), {}, L.ERR_STRIDE),
    (dict(bias_stride=-4), {}, L.ERR_STRIDE),
    (dict(allowed_stride=-4), {}, L.ERR_STRIDE),
    ({}, dict(x=P + 1), L.ERR_ALIGNMENT),
    ({}, dict(out=P + 2, out_dtype=L.DT_F32), L.ERR_ALIGNMENT),
    ({}, dict(idx=P + 4), L.ERR_ALIGNMENT),
    ({}, dict(val=P + 2), L.ERR_ALIGNMENT),
    (dict(ids=P + 2), {}, L.ERR_ALIGNMENT),
    (dict(lengths=P + 1), {}, L.ERR_ALIGNMENT),
    (dict(bias=P + 2), {}, L.ERR_ALIGNMENT),
    (dict(allowed=P + 2), {}, L.ERR_ALIGNMENT),
    (dict(allowed_words=700), dict(MANY, ws=None), L.ERR_WORKSPACE),
    (dict(allowed_words=700), dict(MANY, ws_bytes=200 * 2 * 16 * 8 - 1), L.ERR_WORKSPACE),
    (dict(allowed_words=700), dict(MANY, ws=P + 4), L.ERR_ALIGNMENT),
])
def test_the_entry_point_refuses(rules, kw, code):
    assert adjust(rules, **kw) == code


def test_workspace_bytes():
    def need(M, N, tokens=1, ids=8, bias=4):
        c = L.LogitRules(ids=P, max_ids=ids, repetition=P, bias_ids=P, bias=P, n_bias=bias)
        return L.lib().spectra_adjust_logits_workspace_bytes(ctypes.addressof(c), M, N, L.DT_BF16, tokens)

    assert need(200, 20000) == 200 * 2 * 16 * 8 and need(200, 20000, tokens=0) == 0
    assert need(148, 20000) == 0 and need(149, 20000) > 0 and need(296, 100) == 0 and need(297, 100) > 0
    assert need(200, 20000, ids=6000) == 0 and need(200, 300000) == 0  # lists and rows that one kernel takes
    assert L.lib().spectra_adjust_logits_workspace_bytes(None, 200, 20000, L.DT_BF16, 1) == 0


def test_no_rows_is_no_launch():
    assert adjust(M=0) == L.OK
    assert L.lib().spectra_adjust_logits(None, P, 1, 9, 1, 9, 0, P, 1, 9, None, None, None, 0, None) == L.ERR_NULL_POINTER


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


@pytest.mark.parametrize("kw,err", [
    ({}, ValueError),
    (dict(repetition=1.1), ValueError),                        # penalties of nothing
    (dict(lengths=i32(2)), ValueError),
    (dict(bias_ids=i32(2, 3)), ValueError),
    (dict(bias=torch.zeros(2, 3)), ValueError),
    (dict(ids=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
    (dict(ids=i32(2, 3)), RuntimeError),                       # on the CPU
])
def test_rules_refuse(kw, err):
    with pytest.raises(err):
        LG.LogitRules(**kw)


def test_constants_match_the_header():
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "spectra_b200.h").read_text()
    for name, value in (("MAX_RULE_IDS", L.MAX_RULE_IDS), ("MAX_RULE_BIASES", L.MAX_RULE_BIASES),
                        ("MAX_LISTED_BLOCKS", L.MAX_LISTED_BLOCKS), ("MAX_INDEXED_BLOCKS", L.MAX_INDEXED_BLOCKS),
                        ("MAX_POSITION_AXES", L.MAX_POSITION_AXES)):
        assert f"#define SPECTRA_{name} {value}\n" in text


def test_views_of_one_buffer_beside_each_other_do_not_overlap():
    buf = torch.zeros(4, 64)
    assert not LG._overlap(buf[:, :32], buf[:, 32:]) and not LG._overlap(buf[:, 40:], buf[:, :40])
    assert LG._overlap(buf[:, :33], buf[:, 32:]) and LG._overlap(buf, buf[1:]) and LG._overlap(buf[:, 3:9], buf[:, 8:20])
    assert not LG._overlap(buf[:2], buf[2:]) and not LG._overlap(buf[:0], buf)
    assert LG._overlap(buf, buf.view(8, 32))


def test_the_oracle_by_hand():
    x, t = R.adjust([2.0, -2.0, 1.0, 4.0, 0.5], ids=[0, 1, 1, 0], prompt=2, repetition=2.0, frequency=0.25, presence=0.5,
                    biases=[(4, 1.0), (4, 9.0), (-1, 5.0), (7, 1.0)], allowed=[True, True, True, False, True])
    assert x.tolist() == [0.25, -4.75, 1.0, -np.inf, 9.5] and t == 4
    assert R.adjust([1.0, 3.0, 3.0])[1] == 1 and R.adjust([1.0], allowed=[False])[1] == -1
    assert R.adjust([1.0, np.nan, np.nan])[1] == 1 and R.adjust([5.0, 6.0], offset=10)[1] == 11
