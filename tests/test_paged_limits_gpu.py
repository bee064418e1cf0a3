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
