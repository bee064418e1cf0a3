"""Root mean square error of fp16 attention over lists, loud keys and values,
against 64 bits.

A rounding to 11 bits is off by 2.04e-4 of the number, root mean square (see
tests/test_paged_precision_gpu.py).  Rounded are the values and the result;
the weights are two operands, 22 bits.  Two independent roundings make s =
2.04e-4 sqrt(2) of the result's size, also where the terms of a sum cancel: N
terms of random sign have the size of sqrt(N) of them, and their errors too.
That is an expected value; what a sample shows scatters about it.  Squared
errors w^2 e^2 of variance at most 2 s^4 w^4, alike over all rows of a feature
of a key/value head (they share the values' errors), with W_c the sum of w^2
over such a column: the mean square is s^2 (1 +- sqrt(2 sum W_c^2) / sum W_c),
and three of these deviations are allowed."""
import numpy as np
import pytest
import torch

from oracle import blocks as B
from oracle import paged as R
from spectra_b200 import paged as PG
from tests.test_paged_gpu import DEV, Step, draw
from tests.test_paged_precision_gpu import loud_fill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [0.0, 30.0, 300.0])
@pytest.mark.parametrize("dim,heads,kv_heads", [(32, 8, 2), (64, 8, 2), (96, 4, 2), (128, 8, 1), (128, 12, 1), (256, 4, 2)])
def test_fp16_lists(cap, dim, heads, kv_heads):
    st = Step([700, 300, 90], [4, 1, 3], heads, kv_heads, dim, 32, "f16", seed=71)
    loud_fill(st)
    q = draw((st.total, heads, dim), 72, "f16", 3.0).to(DEV)
    lists = torch.tensor([0, 1, 2, 5, 7, 8, 14, 20, 21], dtype=torch.int32, device=DEV).expand(st.total, kv_heads, 9)
    out = PG.paged_attention(q, st.cache, st.batch, blocks=lists, block_size=32, softcap=cap).cpu().double().numpy()
    err, columns = 0.0, []
    for b, n in enumerate(st.lens):
        rows = slice(st.first[b], st.first[b + 1])
        kv, held, steps = st.ref.values(st.tables[b], n)
        see = held & B.listed(lists[0, 0].tolist(), n, 32)
        want, _, _ = R.attention(q[rows].cpu().double().numpy(), kv[0], kv[1], see, steps, st.positions(b), dim ** -0.5, softcap=cap)
        err += ((out[rows] - want) ** 2).sum()
        columns.append((want ** 2).reshape(-1, kv_heads, heads // kv_heads, dim).sum((0, 2)).ravel())
    w = np.concatenate(columns)
    bound = 2.04e-4 * 2 ** 0.5 * (1 + 3 * (2 * (w ** 2).sum()) ** 0.5 / w.sum()) ** 0.5
    got = (err / w.sum()) ** 0.5
    assert got <= bound, f"{got:.2e} of {bound:.2e}"
