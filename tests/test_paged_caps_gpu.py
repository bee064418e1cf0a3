"""Caps far from the scores' size: the root mean square error against 64 bits.

Bound: each rounding to 11 bits (keys, values, weights, an fp16 output) is off by 2^-12 / sqrt(3) of
its operand, 1.4e-4; a score of up to about 5 is then off by 7e-4, and so is its weight.  Together
well below 2^-9 of the result; a bf16 output adds 2^-9 / sqrt(3): 2^-8."""
import numpy as np
import pytest
import torch

from oracle import paged as R
from spectra_b200 import paged as PG
from tests.test_paged_gpu import DEV, Step, draw, f32

pytestmark = pytest.mark.gpu


def rms_check(st, q, out, keys=None, **kw):
    """``keys``: the type that the reference's keys are rounded to first."""
    assert torch.isfinite(out).all()
    kw.setdefault("scale", st.dim ** -0.5)
    qd, od = q.cpu().double().numpy(), out.cpu().double().numpy()
    want = np.zeros_like(od)
    for b, n in enumerate(st.lens):
        rows = slice(st.first[b], st.first[b + 1])
        kv, held, steps = st.ref.values(st.tables[b], n)
        if keys is not None:
            kv[0] = kv[0].astype(keys)
        want[rows], _, _ = R.attention(qd[rows], kv[0], kv[1], held, steps, st.positions(b), **kw)
    err = np.sqrt(((od - want) ** 2).sum() / (want ** 2).sum())
    bound = 2.0 ** (-8 if out.dtype == torch.bfloat16 else -9)
    assert err <= bound, f"{err:.2e} of {bound:.2e}"


@pytest.mark.parametrize("cap", [3.0, 50.0, 1e4, 1e6, 1e12, 3e38])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dim,lens,news", [(64, [300, 77, 150], [1, 1, 1]), (128, [300, 77, 150], [3, 2, 1]),
                                           (64, [300, 277], [200, 130]), (128, [500, 130], [140, 130]),
                                           (256, [300, 400], [300, 290])])
def test_caps_up_to_the_largest(cap, bias, dim, lens, news):
    st = Step(lens, news, 4, 2, dim, 32, "f16", seed=41)
    st.fill(spread=0.5)
    q = (draw((st.total, 4, dim), 42, "f16", 0.0) * 4).to(DEV)
    slopes = np.exp2(-2.0 * np.arange(1, 5)).astype(np.float32) if bias else None
    out = PG.paged_attention(q, st.cache, st.batch, softcap=cap,
                             alibi_slopes=None if slopes is None else torch.from_numpy(slopes).to(DEV))
    rms_check(st, q, out, softcap=cap, slopes=slopes)


@pytest.mark.parametrize("dim,news", [(64, [1, 1]), (128, [2, 5]), (64, [150, 200]), (128, [300, 129])])
@pytest.mark.parametrize("cap,loud", [(1e-3, 1.0), (1e-30, 1.0), (1e-42, 1.0), (30.0, 1e12), (30.0, 1e25)])
def test_caps_far_below_the_scores(dim, news, cap, loud):
    """Scores at the cap, and keys of zeros, whose score stays 0.  Of loud queries a score's sign is all
    that is left, and the prompts' keys, rounded to fp16, give some of the smallest the other one: their
    reference has the rounded keys (the rounding alone makes 4e-3 to 8e-3)."""
    st = Step([300, 200], news, 4, 2, dim, 32, "bf16", seed=43)
    st.fill()
    for b in range(2):
        st.ref.append(st.tables[b], np.arange(64, 160), np.zeros((96, 2, dim), np.float32),
                      f32(draw((96, 2, dim), 44 + b, "bf16")))
    st.upload()
    q = (draw((st.total, 4, dim), 46, "bf16").float() * loud).to(torch.bfloat16).to(DEV)
    rms_check(st, q, PG.paged_attention(q, st.cache, st.batch, softcap=cap),
              keys=np.float16 if loud > 1.0 and max(news) > 48 else None, softcap=cap)
