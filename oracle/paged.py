"""CPU oracle for the paged INT4 KV cache (numpy): rotation, quantiser, the
pool's byte layout and attention over it.

TEST INFRASTRUCTURE ONLY, like the rest of this package.  The arithmetic of
the append (rotation and codes) is restated in fp32, operation by operation;
the attention is the definition in fp64.
"""
from __future__ import annotations

import numpy as np

GROUP = 32


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [T, H, D] fp32, cos/sin [T, rotary / 2] fp32 (the rows of the tokens' positions)."""
    x = np.asarray(x, np.float32).copy()
    half = cos.shape[1]
    if half == 0:
        return x
    lo, hi = (np.arange(half) * 2, np.arange(half) * 2 + 1) if interleaved else (np.arange(half), np.arange(half) + half)
    a, b, c, s = x[..., lo].copy(), x[..., hi].copy(), cos[:, None], sin[:, None]
    with np.errstate(invalid="ignore", over="ignore"):
        x[..., lo] = a * c - b * s
        x[..., hi] = b * c + a * s
    return x


def quantize(k: np.ndarray, v: np.ndarray):
    """fp32 keys and values [..., D] -> (codes u8 [..., 2, D], scales fp16 [..., 2, G], zeros u8 [..., 2, G])."""
    x = np.stack([k, v], -2).astype(np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        lo = np.minimum(np.fmin.reduce(g, -1), np.float32(0))
        hi = np.maximum(np.fmax.reduce(g, -1), np.float32(0))
        ok = np.isfinite(g).all(-1) & (hi - lo <= np.float32(65472))
        ok = np.broadcast_to(ok.all(-2, keepdims=True), ok.shape)  # key and value group together
        s = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
        s32 = s.astype(np.float32)
        r = np.where(s32 > 0, np.float32(1) / s32, np.float32(0)).astype(np.float32)
        z = np.minimum(np.rint(-lo * r), np.float32(15))
        q = np.clip(np.rint(g * r[..., None]) + z[..., None], 0, 15)
    s = np.where(ok, s, np.float16(0))
    s[..., 0, :] = np.where(ok[..., 0, :], s[..., 0, :], np.float16(np.nan))
    q = np.where(ok[..., None], q, 0).astype(np.uint8).reshape(x.shape)
    return q, s, np.where(ok, z, 0).astype(np.uint8)


class Pool:
    """A pool as plain arrays: codes [pages, H, page, 2, D], scales and zeros [pages, H, page, 2, G]."""

    def __init__(self, pages: int, heads: int, dim: int, page: int):
        self.page, self.dim = page, dim
        self.codes = np.zeros((pages, heads, page, 2, dim), np.uint8)
        self.scales = np.zeros((pages, heads, page, 2, dim // GROUP), np.float16)
        self.zeros = np.zeros((pages, heads, page, 2, dim // GROUP), np.uint8)

    def to_bytes(self) -> np.ndarray:
        """[pages, H, page / 16, 608 G] in the layout of include/spectra_b200.h."""
        n, H, P, _, D = self.codes.shape
        G, T = D // GROUP, P // 16
        c = self.codes.reshape(n, H, T, 2, 8, 2, D)                          # tile, block, token
        b = (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(n, H, T, 2, 8, 2, G, 16)
        key = b[:, :, :, :, :, 0].reshape(n, H, T, 2, 8, G, 4, 4).transpose(0, 1, 2, 3, 4, 6, 5, 7)
        val = b[:, :, :, :, :, 1].reshape(n, H, T, 2, 4, 2, G, 8, 2).transpose(0, 1, 2, 3, 7, 4, 6, 5, 8)
        s = self.scales.reshape(n, H, T, 8, 2, 2, G)
        z = self.zeros.reshape(n, H, T, 8, 2, 2, G)
        flat = lambda a: np.ascontiguousarray(a).view(np.uint8).reshape(n, H, T, -1)  # noqa: E731
        return np.concatenate([flat(key), flat(val), flat(s[..., 0, :]), flat(s[..., 1, :].swapaxes(-1, -2)),
                               flat(z[..., 0, :]), flat(z[..., 1, :].swapaxes(-1, -2))], -1)

    def append(self, table, pos, k, v):
        """Tokens at positions pos [n] of one sequence; k, v fp32 [n, H, D]."""
        q, s, z = quantize(k, v)
        for i, p in enumerate(pos):
            page = int(table[p // self.page])
            if p < 0 or not 0 <= page < self.codes.shape[0]:
                continue
            at = (page, slice(None), p % self.page)
            self.codes[at], self.scales[at], self.zeros[at] = q[i], s[i], z[i]

    def values(self, table, n):
        """fp64 keys and values [2, n, H, D] of a sequence's first n tokens, which of them a page holds, and the
        keys' scales [n, H, G]."""
        H, G = self.codes.shape[1], self.dim // GROUP
        out, held, steps = np.zeros((2, n, H, self.dim)), np.zeros(n, bool), np.zeros((n, H, G))
        for p in range(n):
            page = int(table[p // self.page])
            if not 0 <= page < self.codes.shape[0]:
                continue
            at = (page, slice(None), p % self.page)
            q = self.codes[at].astype(np.float64).reshape(H, 2, G, GROUP)
            out[:, p] = ((q - self.zeros[at][..., None]) * self.scales[at].astype(np.float64)[..., None]).reshape(
                H, 2, self.dim).swapaxes(0, 1)
            held[p], steps[p] = True, self.scales[at][:, 0]
        return out, held, steps


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, held: np.ndarray, steps: np.ndarray, pos, scale: float,
              causal=True, window=0, softcap=0.0, slopes=None):
    """One sequence: q [m, Hq, D] at positions pos [m]; k, v [n, H, D] fp64.
    Returns out, spread = sum p |v| (what a relative error of the weights or
    the values is multiplied by), and the sizes [2, m, Hq] that the error of a
    score scales with: the largest sum |q| |k| of a key that the row sees, and
    the largest sum over its groups of scale times sum |q|."""
    m, Hq, D = q.shape
    n, H, _ = k.shape
    r = Hq // H
    out, spread, size = np.zeros((m, Hq, D)), np.zeros((m, Hq, D)), np.zeros((2, m, Hq))
    idx = np.arange(n)
    for i in range(m):
        if pos[i] < 0:
            continue
        see = held.copy()
        if causal:
            see &= idx <= pos[i]
        if window:
            see &= idx > max(int(pos[i]) - int(window), -1)  # (any window: numpy's integers have 64 bits)
        if not see.any():
            continue
        for h in range(Hq):
            K, V = k[see, h // r], v[see, h // r]
            with np.errstate(invalid="ignore", over="ignore"):
                t = scale * (K @ q[i, h])
                if softcap:
                    t = softcap * np.tanh(t / softcap)
                if slopes is not None:
                    t = t + slopes[h] * (idx[see] - pos[i])
                p = np.exp(t - np.max(t))
                p /= p.sum()
                out[i, h], spread[i, h] = p @ V, p @ np.abs(V)
                absq = np.abs(q[i, h])
                size[0, i, h] = np.max(np.abs(K) @ absq)
                size[1, i, h] = np.max(steps[see, h // r] @ absq.reshape(-1, GROUP).sum(-1))
    return out, spread, size
