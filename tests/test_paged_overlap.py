"""Outputs given to the paged operators: refused where they share an element
with an input, taken where they only lie between its rows."""
import random

import pytest
import torch

from spectra_b200 import paged as PG


def elements(t):
    i = torch.arange(t.shape[0])[:, None, None] * t.stride(0) + torch.arange(t.shape[1])[:, None] * t.stride(1)
    return set((t.storage_offset() + i + torch.arange(t.shape[2])).flatten().tolist())


def test_overlap_is_exact():
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(3000):
        T, D = rng.randint(1, 5), rng.choice([4, 8])
        buf = torch.zeros(600, dtype=torch.float16)

        def view():
            H = rng.randint(1, 3)
            hs = rng.choice([D, D, 2 * D, D + 3, 0])
            ts = rng.choice([H * D, 6 * D, 6 * D, 40, 1, 0])
            return buf.as_strided((rng.randint(1, T), H, D), (ts, hs, 1), rng.randint(0, 300))

        a, b = view(), view()
        want = bool(elements(a) & elements(b))
        assert PG._overlap(a, b) == want and PG._overlap(b, a) == want, (a.shape, a.stride(), b.shape, b.stride())
        seen[want] += 1
    assert min(seen) > 300
    c = torch.zeros(3, 2, 8)
    assert not PG._overlap(c, torch.zeros(3, 2, 8)) and not PG._overlap(c[:0], c)


@pytest.mark.gpu
def test_outputs_that_overlap_inputs():
    from tests.test_paged_gpu import DEV, Step, draw

    st = Step([40, 30], [40, 30], 4, 2, 64, 16, "bf16", seed=51)
    st.fill()
    T = st.total
    wide = draw((T, 16, 64), 52, "bf16").to(DEV)
    q, k, v, free = wide[:, :4], wide[:, 4:6], wide[:, 6:8], wide[:, 8:12]
    want = PG.paged_kv_append(st.cache, st.batch, k, v, q=q)
    for out in (q, k.reshape(T, 2, 64)[:, :1].expand(T, 4, 64), wide[:, 1:5], wide[:, 2:6], wide[:, 3:7], wide[:, 7:11],
                torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(T, 4, 64)):
        with pytest.raises(ValueError, match="out must not"):
            PG.paged_kv_append(st.cache, st.batch, k, v, q=q, out=out)
    assert torch.equal(PG.paged_kv_append(st.cache, st.batch, k, v, q=q, out=free), want)  # between the inputs' rows
    assert torch.equal(free, want)

    want = PG.paged_attention(q, st.cache, st.batch)
    for out in (wide[:, 1:5], wide[:, 3:7], wide[1:, :4].new_zeros(1, 4, 64).expand(T, 4, 64)):
        with pytest.raises(ValueError, match="out must not"):
            PG.paged_attention(q, st.cache, st.batch, out=out)
    flat = torch.zeros((T + 1) * 4 * 64, dtype=torch.bfloat16, device=DEV)
    moved = flat[:T * 256].view(T, 4, 64)
    with pytest.raises(ValueError, match="unless it is q"):
        PG.paged_attention(moved, st.cache, st.batch, out=flat[256:].view(T, 4, 64))
    assert torch.equal(PG.paged_attention(q, st.cache, st.batch, out=free), want)
    assert torch.equal(PG.paged_attention(q, st.cache, st.batch, out=q), want)  # in place
    assert torch.equal(q, want)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", [([9000, 3, 7000], [1, 1, 1]), ([900], [300]), ([300, 290, 80], [200, 1, 33])])
def test_attention_in_place_of_split_sequences(lens, news):
    from tests.test_paged_gpu import DEV, Step, draw

    st = Step(lens, news, 8, 2, 128, 16, "bf16", seed=53)
    st.fill()
    q = draw((st.total, 8, 128), 54, "bf16").to(DEV)
    want = PG.paged_attention(q, st.cache, st.batch)
    assert PG.paged_attention(q, st.cache, st.batch, out=q) is q
    assert torch.equal(q, want)
