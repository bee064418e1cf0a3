"""Attention over lists with more or fewer segments (tokens times key/value
heads) than the GPU holds at once with three and with four CTAs an SM: the
kernel that is chosen, and the turns that its CTAs take."""
import numpy as np
import pytest
import torch

from spectra_b200 import paged as PG
from tests.test_paged_blocks_gpu import attend, random_lists
from tests.test_paged_gpu import DEV, Step, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per_sm", [3, 4, 9])
@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("dim,heads,dt,case", [(32, 4, "bf16", "plain"), (64, 4, "f16", "cap"), (64, 11, "bf16", "all"), (32, 1, "f16", "window")])
def test_segments_about_what_the_gpu_holds(per_sm, more, dim, heads, dt, case):
    n = per_sm * torch.cuda.get_device_properties(0).multi_processor_count + more
    if n * -(-heads // 8) % 7 == 0:
        n += 1  # (the last turn is not full)
    st = Step([(13 * i) % 200 + 1 for i in range(n)], [1] * n, heads, 1, dim, 32, dt, seed=per_sm)
    rng = np.random.default_rng(dim)
    st.ref.codes[:] = rng.integers(0, 16, st.ref.codes.shape, np.uint8)
    st.ref.scales[:] = rng.uniform(0.02, 0.4, st.ref.scales.shape).astype(np.float16)
    st.ref.zeros[:] = rng.integers(0, 16, st.ref.zeros.shape, np.uint8)
    st.upload()
    q = draw((n, heads, dim), 95, dt).to(DEV)
    lists = random_lists(st, 4, 32, per_sm)
    out = attend(st, q, lists, 32, case)
    kw = dict(plain={}, cap=dict(softcap=5.0), window=dict(window=100), all=None)[case]
    if kw is not None:
        assert torch.equal(out, PG.paged_attention(q, st.cache, st.batch, blocks=lists, block_size=32, **kw))
