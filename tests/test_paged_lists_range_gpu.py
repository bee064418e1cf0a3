"""Attention over lists where a row sees a small part of the blocks listed for
it (blocks far larger than the sequence, windows that begin inside a block,
positions inside one): results as the oracle has them, and no time spent on
what no row sees."""
import numpy as np
import pytest
import torch

from spectra_b200 import kernels as SK
from spectra_b200 import paged as PG
from tests.test_paged_blocks_gpu import attend, check_lists, random_lists
from tests.test_paged_gpu import DEV, Step, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [32, 1024, 65536])
@pytest.mark.parametrize("dim,dt,page", [(64, "bf16", 16), (128, "f16", 64)])
def test_blocks_far_larger_than_the_sequences(block, dim, dt, page):
    st = Step([100, 1, 33, 0, 700, 64], [1] * 6, 8, 2, dim, page, dt, seed=block % 97)
    st.fill()
    q = draw((6, 8, dim), 90, dt).to(DEV)
    every = torch.arange(-(-700 // block), dtype=torch.int32, device=DEV).expand(6, 2, -1)
    st.check(q, attend(st, q, every, block))


@pytest.mark.parametrize("case", ["plain", "full", "window", "all"])
@pytest.mark.parametrize("block", [512, 4096])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (20, 1)])
def test_windows_and_positions_inside_a_block(case, block, heads, kv_heads):
    """Several rows of a sequence: the keys of each begin and end in other units."""
    st = Step([1500, 600, 513, 4200], [40, 3, 1, 7], heads, kv_heads, 64, 32, "bf16", seed=block)
    st.fill()
    attend(st, draw((st.total, heads, 64), 91, "bf16").to(DEV), random_lists(st, 4, block, 8), block, case)


@pytest.mark.parametrize("case", ["plain", "window", "full"])
@pytest.mark.parametrize("block", [256, 16384])
def test_one_row_in_pieces(case, block):
    """One segment, which many CTAs share; all but a few units of its last block lie past the sequence."""
    st = Step([20000], [1], 4, 1, 128, 64, "bf16", seed=6)
    st.fill()
    q = draw((1, 4, 128), 92, "bf16").to(DEV)
    n = -(-20000 // block)
    lists = torch.arange(n, dtype=torch.int32, device=DEV)[None, None]
    a = attend(st, q, lists, block, case)
    for _ in range(3):
        b = PG.paged_attention(q, st.cache, st.batch, blocks=lists, block_size=block, causal=case != "full",
                               window=100 if case == "window" else 0)
        assert torch.equal(a, b)
    assert SK.device_timeouts() == 0


def test_positions_past_the_bound_and_a_window_that_begins_there():
    """Tokens whose position passes max_len see what is held before it, and nothing where their window begins past it."""
    st = Step([300, 260], [80, 4], 4, 2, 64, 32, "bf16", seed=5, max_len=250)
    st.fill()
    q = draw((84, 4, 64), 93, "bf16").to(DEV)
    lists = torch.arange(3, dtype=torch.int32, device=DEV).expand(84, 2, 3)
    for block in (128, 1024):
        kw = dict(window=30)
        out = PG.paged_attention(q, st.cache, st.batch, blocks=lists, block_size=block, **kw)
        check_lists(st, q, out, lists, block, None, 250, **kw)
        assert not out[70].any() and not out[79].any()  # positions 290 and 299


@pytest.mark.parametrize("what", ["past the sequence", "before the window"])
def test_time_does_not_grow_with_the_part_of_a_block_that_no_row_sees(what):
    """512 segments over the same 100 keys (four units) in blocks of 128 and of far more: a kernel that read whole
    blocks would take over a hundred times as long."""
    n, dim, page = 64, 128, 64
    length, window = (100, 0) if what == "past the sequence" else (8192, 100)
    each = -(-length // page)
    tables = torch.arange(n * each, dtype=torch.int32, device=DEV).reshape(n, each)
    cache = PG.PagedKVCache(n * each, 8, dim, page_size=page)
    batch = PG.TokenBatch(tables, torch.full((n,), length, dtype=torch.int32, device=DEV))
    q = draw((n, 8, dim), 94, "bf16").to(DEV)

    def median(block):
        first = max(0, length - 100) // block
        lists = torch.arange(first, first + 2, dtype=torch.int32, device=DEV).expand(n, 8, 2)
        for _ in range(3):
            PG.paged_attention(q, cache, batch, blocks=lists, block_size=block, window=window)
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                PG.paged_attention(q, cache, batch, blocks=lists, block_size=block, window=window)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return float(np.median(times))

    small, large = median(128), median(65536 if what == "past the sequence" else 8192)
    assert large < 3 * small, f"{large:.3f} ms with large blocks, {small:.3f} with small ones"
