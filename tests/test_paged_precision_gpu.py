"""Root mean square error of fp16 results over loud keys and values, against 64 bits.

A rounding to 11 bits is off by 2.04e-4 of the number, root mean square (2^-11 / sqrt(12) over the mean of
[1, 2)'s squares' inverse: 2^-11 * 0.2887 * 1.445).  Weights and the result are rounded: 2.9e-4 together.
Prompts with heads of up to 64: their keys and values are exact."""
import numpy as np
import pytest
import torch

from oracle import paged as R
from spectra_b200 import paged as PG
from tests.test_paged_gpu import DEV, MASKS, Step, draw

pytestmark = pytest.mark.gpu


def loud_fill(st):
    """Keys with features of 7, values of 3 times the rest's size."""
    for b, n in enumerate(st.lens):
        k, v = (draw((n, st.kv_heads, st.dim), 100 * st.seed + 2 * b + i, "f16", s).float().numpy() for i, s in ((0, 6.0), (1, 2.0)))
        st.ref.append(st.tables[b], np.arange(n), k, v)
    return st.upload()


PROMPTS = [(64, 4, 4, [900], [400]), (64, 4, 2, [600, 700], [500, 300]), (32, 8, 2, [500, 300], [300, 300]),
           (64, 16, 2, [700, 300, 90], [60, 200, 90])]


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("dim,heads,kv_heads,lens,news", PROMPTS)
def test_fp16_prompts(mask, dim, heads, kv_heads, lens, news):
    st = Step(lens, news, heads, kv_heads, dim, 32, "f16", seed=71)
    loud_fill(st)
    q = draw((st.total, heads, dim), 72, "f16", 3.0).to(DEV)
    kw = dict(MASKS[mask])
    slopes = None
    if kw.pop("alibi", False):
        slopes = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32)
    out = PG.paged_attention(q, st.cache, st.batch, alibi_slopes=None if slopes is None else torch.from_numpy(slopes).to(DEV), **kw)
    err = size = 0.0
    for b, n in enumerate(lens):
        rows = slice(st.first[b], st.first[b + 1])
        kv, held, steps = st.ref.values(st.tables[b], n)
        want, _, _ = R.attention(q[rows].cpu().double().numpy(), kv[0], kv[1], held, steps, st.positions(b), dim ** -0.5,
                                 slopes=slopes, **kw)
        err, size = err + ((out[rows].cpu().double().numpy() - want) ** 2).sum(), size + (want ** 2).sum()
    bound = 2.9e-4
    assert (err / size) ** 0.5 <= bound, f"{(err / size) ** 0.5:.2e} of {bound:.1e}"
