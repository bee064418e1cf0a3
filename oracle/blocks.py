"""CPU oracle for the block index of the paged cache, the choice of blocks and
what a list of blocks leaves of the keys (numpy).

TEST INFRASTRUCTURE ONLY, like the rest of this package.  Keys are the fp64
values of ``oracle.paged.Pool.values``; every step here is exact.
"""
from __future__ import annotations

import numpy as np


def step(most: float) -> float:
    """The least power of two, from 2^-126 on, whose 127-fold reaches ``most``; 1 for 0."""
    if most == 0:
        return 1.0
    e = max(int(np.floor(np.log2(most))) - 9, -126)
    while 127 * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def bounds(keys: np.ndarray):
    """One block's keys [n, D] -> codes int8 [2, D] (largest, smallest), scale."""
    if not np.isfinite(keys).all():
        return np.zeros((2, keys.shape[1]), np.int8), np.inf
    hi, lo = keys.max(0), keys.min(0)
    s = step(max(np.abs(hi).max(), np.abs(lo).max()))
    return np.stack([np.ceil(hi / s), np.floor(lo / s)]).astype(np.int8), s


def query_codes(q: np.ndarray) -> np.ndarray:
    """Queries [r, D] fp64 -> integers [r, D], each row in a step of its own."""
    out = np.zeros(q.shape, np.int64)
    for i, row in enumerate(q):
        if np.isfinite(row).all():
            out[i] = np.rint(row / step(np.abs(row).max()))
    return out


def scores(q: np.ndarray, codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """q [r, D] of one key/value head, codes [n, 2, D], scales [n] -> [n]."""
    c = query_codes(q)
    k = codes.astype(np.int64)
    s = (np.maximum(c, 0) @ k[:, 0].T + np.minimum(c, 0) @ k[:, 1].T).max(0).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(np.isinf(scales), np.inf, s * scales)


def select(q, codes, scales, held, n: int, count: int, first: int, last: int) -> list:
    """Blocks of one token and key/value head: q [r, D]; codes, scales, held of its n blocks."""
    always = [j for j in range(n) if (j < first or j >= n - last) and held[j]]
    rest = np.array([j for j in range(first, n - last) if held[j]], np.int64)
    free = count - len(always)
    if len(always) + len(rest) > count:
        s = scores(q, codes[rest], scales[rest])
        rest = rest[np.argsort(-s, kind="stable")[:free]]
    return sorted(always + rest.tolist())


def listed(blocks, n: int, block: int) -> np.ndarray:
    """Which of a sequence's n tokens a list names: entries above all before them."""
    see, top = np.zeros(n, bool), -1
    for b in blocks:
        if b > top:
            see[min(n, int(b) * block):min(n, (int(b) + 1) * block)] = True
            top = int(b)
    return see
