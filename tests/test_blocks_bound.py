"""What the score of the choice of blocks is: for every query head an upper
bound of the head's rounded codes times the keys of the block, each head in a
step of its own.  By the oracle, which the kernels equal (no GPU)."""
import numpy as np
import pytest

from oracle import blocks as B


def draw(seed, blocks=20, size=32, dim=64, heads=4):
    rng = np.random.default_rng(seed)
    steps = rng.uniform(0.01, 2.0, (blocks, size, dim // 32)).astype(np.float16).astype(np.float64)
    keys = (rng.integers(0, 16, (blocks, size, dim)) - rng.integers(0, 16, (blocks, size, dim // 32)).repeat(32, -1)) * steps.repeat(32, -1)
    q = rng.normal(size=(heads, dim)) * np.exp(rng.normal(size=(heads, 1)) * 3)
    codes, scales = zip(*(B.bounds(k) for k in keys))
    return q, keys, np.stack(codes), np.array(scales)


@pytest.mark.parametrize("seed", range(5))
def test_the_score_bounds_the_codes_times_every_key(seed):
    q, keys, codes, scales = draw(seed)
    c = B.query_codes(q)
    assert ((64 <= np.abs(c).max(-1)) & (np.abs(c).max(-1) <= 127)).all()
    products = np.einsum("hd,bnd->bhn", c.astype(np.float64), keys)
    # (keys have 15 bits and codes 7: the products and their sums are exact)
    assert (B.scores(q, codes, scales) >= products.max((1, 2))).all()
    alone = np.stack([B.scores(q[h:h + 1], codes, scales) for h in range(len(q))])
    assert (alone >= products.max(2).T).all() and np.array_equal(alone.max(0), B.scores(q, codes, scales))


def test_a_heads_step_does_not_count_and_the_score_is_no_bound_of_q_times_k():
    q, keys, codes, scales = draw(9)
    want = B.scores(q, codes, scales)
    for h in range(len(q)):  # a head times a power of two votes as before
        louder = q.copy()
        louder[h] *= 2.0**40
        assert np.array_equal(B.scores(louder, codes, scales), want)
    loud = q * 2.0**40
    assert (np.einsum("hd,bnd->bhn", loud, keys).max((1, 2)) > B.scores(loud, codes, scales)).any()
