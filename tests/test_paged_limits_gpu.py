"""The paged INT4 KV cache at the ends of its arguments' ranges."""
import pytest
import torch

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
