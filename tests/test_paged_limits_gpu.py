"""The paged INT4 KV cache at the ends of its arguments' ranges."""
import numpy as np
import pytest
import torch

from tests.test_paged_caps_gpu import rms_check
from tests.test_paged_gpu import DEV, Step, draw, run_masked
from spectra_b200 import paged as PG

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**40, 2**64 + 7, 300, 1])
@pytest.mark.parametrize("dim,lens,news", [
    (64, [40, 200, 3, 6], [9, 9, 9, 9]),             # sequences 2 and 3 hold fewer tokens than are new: padding
    (128, [5, 200, 1, 0], [8, 3, 6, 4]),
    (64, [150, 60, 1], [200, 200, 200]),             # the same with prompts
    (256, [130, 300, 40], [140, 65, 150]),
    (128, [90], [300]),                              # one prompt, its keys split
])
def test_attention_window_of_any_size_with_padding(window, dim, lens, news):
    st = Step(lens, news, 4, 2, dim, 16, "bf16", seed=21)
    st.fill()
    q = draw((st.total, 4, dim), 22, "bf16").to(DEV)
    for causal in (True, False):
        out = run_masked(st, q, "plain", window=window, causal=causal)
        if window >= 300:  # none of these rows is cut by it
            assert torch.equal(out, PG.paged_attention(q, st.cache, st.batch, causal=causal))


@pytest.mark.parametrize("dim,max_q,news", [
    (64, 2, [5, 2, 1]), (128, 1, [40, 1, 1]), (256, 3, [9, 2, 200]),   # few rows
    (64, 100, [300, 30, 7]), (128, 64, [129, 70, 1]), (256, 200, [300, 130, 2]),   # prompts, both kernels
    (128, 60, [400, 350, 300]),
])
def test_attention_rows_past_max_q_are_zero(dim, max_q, news):
    st = Step([450, 360, 310], news, 4, 2, dim, 16, "bf16", seed=23, uniform=False)
    st.fill()
    q = draw((st.total, 4, dim), 24, "bf16").to(DEV)
    good = run_masked(st, q, "plain")
    batch = PG.TokenBatch(st.t_tables, st.t_lens, cu_q=st.batch.cu_q, total=st.total, max_q=max_q)
    out = torch.full_like(q, 7.0)
    PG.paged_attention(q, st.cache, batch, out=out)
    for b, n in enumerate(news):
        past = slice(st.first[b] + min(n, max_q), st.first[b + 1])
        assert not out[past].any()
        out[past] = good[past]
    st.check(q, out)


def test_a_c_caller_s_max_q_does_not_cut_equal_sequences():
    """Without cu_q the rows of a sequence are q_len, whatever max_q says."""
    for n, max_q in ((6, 1), (150, 1), (400, 60)):
        st = Step([500, 470], [n, n], 4, 2, 64, 16, "bf16", seed=25)
        st.fill()
        q = draw((st.total, 4, 64), 26, "bf16").to(DEV)
        st.batch._c.max_q = max_q
        out = torch.full_like(q, 7.0)
        st.check(q, PG.paged_attention(q, st.cache, st.batch, out=out))


@pytest.mark.parametrize("loud", [1e20, 1e30, 1e34])
@pytest.mark.parametrize("dim,lens,news", [(64, [1, 2, 9, 40], [1, 1, 1, 1]), (128, [5, 3], [5, 2]), (64, [150, 140], [150, 130]),
                                           (128, [120, 200], [110, 150]), (256, [300], [300])])
def test_attention_scores_up_to_what_fp32_holds(loud, dim, lens, news):
    """bf16 queries of any size: the key of the highest score takes all the weight, also where every score a row
    sees is far below zero (as of a row that sees one key, half the time)."""
    st = Step(lens, news, 4, 2, dim, 16, "bf16", seed=27)
    st.fill(spread=0.0)
    q = (draw((st.total, 4, dim), 28, "bf16", 0.0).float() * loud).to(torch.bfloat16).to(DEV)
    out, qd = PG.paged_attention(q, st.cache, st.batch).cpu().double().numpy(), q.cpu().double().numpy()
    rows = below = 0
    for b, n in enumerate(lens):
        kv, _, _ = st.ref.values(st.tables[b], n)
        for i, p in enumerate(st.positions(b)):
            for h in range(4):
                t = kv[0][:p + 1, h // 2] @ qd[st.first[b] + i, h]
                order = np.argsort(t)
                # the keys' 11 bits move a product by 2^-11 of its terms' sizes at most
                size = (np.abs(kv[0][:p + 1, h // 2]) @ np.abs(qd[st.first[b] + i, h])).max()
                if p and t[order[-1]] - t[order[-2]] <= 2.0**-9 * size:
                    continue
                want = kv[1][order[-1], h // 2]
                assert (np.abs(out[st.first[b] + i, h] - want) <= (2.0**-8 + 2.0**-10) * np.abs(want)).all(), (b, p, h)
                rows, below = rows + 1, below + (t.max() < 0)
    # (of the inputs: rows that see few keys)
    assert rows > 4 and (below > 0 or min(st.positions(b)[0] for b in range(len(lens))) > 8)


@pytest.mark.parametrize("scale,quiet", [(1e-12, 1.0), (1e-20, 2.0**-60), (1e-30, 2.0**-100), (1e-37, 0.0)])
@pytest.mark.parametrize("dim,lens,news", [(64, [1, 2, 9, 77], [1, 1, 1, 1]), (128, [50, 3], [5, 2]), (64, [150, 140], [150, 130]),
                                           (256, [300], [300])])
def test_attention_scores_that_vanish(scale, quiet, dim, lens, news):
    """Equal weights, and masks that stay masks where a row's factor is 0 in fp32."""
    st = Step(lens, news, 4, 2, dim, 16, "bf16", seed=29)
    st.fill(spread=0.0)
    q = (draw((st.total, 4, dim), 30, "bf16", 0.0).float() * quiet).to(torch.bfloat16).to(DEV)
    for kw in ({}, dict(window=11)):
        rms_check(st, q, PG.paged_attention(q, st.cache, st.batch, scale=scale, **kw), scale=scale, **kw)
