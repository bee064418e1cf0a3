"""The block index of many blocks (the kernel of bulk copies) where keys are
not finite, and with sequences laid out in groups of 128, blocks of sixteen
pieces and a number of heads that is no power of two.  The pool's bytes are
drawn as they are: filling it token by token takes long."""
import numpy as np
import pytest
import torch

from oracle import blocks as B
from spectra_b200 import kernels as SK
from spectra_b200 import paged as PG
from tests.test_paged_blocks_gpu import same
from tests.test_paged_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kv_heads,page,block,batch", [(64, 3, 512, 512, 300), (32, 16, 64, 32, 150), (96, 12, 128, 64, 150),
                                                           (128, 16, 64, 64, 150), (256, 8, 128, 128, 200), (128, 5, 256, 256, 260)])
def test_keys_that_are_not_finite_among_many_blocks(dim, kv_heads, page, block, batch):
    lens = [block + (37 * i) % (3 * block) if i % 7 else 0 for i in range(batch)]
    news = [max(1, n - (11 * i) % 40) for i, n in enumerate(lens)]
    blocks = -(-max(news) // block)
    assert blocks > 1 and blocks * kv_heads * batch > 16 * torch.cuda.get_device_properties(0).multi_processor_count
    st = Step(lens, news, kv_heads, kv_heads, dim, page, "bf16", seed=block)
    rng = np.random.default_rng(dim)
    pages, groups = len(st.ref.codes), dim // 32
    st.ref.codes[:] = rng.integers(0, 16, st.ref.codes.shape, np.uint8)
    st.ref.scales[:] = rng.uniform(0.01, 3.0, st.ref.scales.shape).astype(np.float16)
    st.ref.zeros[:] = rng.integers(0, 16, st.ref.zeros.shape, np.uint8)
    # a few key scales of a page's first, last and some other token, and of values, which do not count
    for i, value in enumerate([np.nan, np.inf, -np.inf] * (pages // 9)):
        at = rng.integers(pages), rng.integers(kv_heads), (0, page - 1, rng.integers(page))[i // 3 % 3]
        st.ref.scales[(*at, int(i % 4 == 3), rng.integers(groups))] = value
    st.upload()
    index = PG.BlockIndex(st.cache, block)
    PG.paged_index_update(index, st.batch)
    codes, scales = np.zeros(index.codes.shape, np.int8), np.zeros(index.scales.shape, np.float32)
    for b, (n, new) in enumerate(zip(lens, news)):
        for j in range(max(0, n - new) // block, n // block):
            p, part = int(st.tables[b, j * block // page]), j % (page // block)
            span = slice(part * block, (part + 1) * block)
            for h in range(kv_heads):
                s = st.ref.scales[p, h, span, 0].astype(np.float64)[..., None]
                q = st.ref.codes[p, h, span, 0].astype(np.float64).reshape(block, groups, 32)
                with np.errstate(invalid="ignore"):
                    keys = (q - st.ref.zeros[p, h, span, 0].astype(np.float64)[..., None]) * s
                codes[p, h, part], scales[p, h, part] = B.bounds(keys.reshape(block, dim))
    assert np.isinf(scales).sum() > 3 and np.isfinite(scales).sum() > 100
    same(index, (codes, scales))
    assert SK.device_timeouts() == 0
