"""Paged INT4 KV cache: rotate-and-append, read back, attention over the codes.

The reference keeps its INT4 cache as one dense tensor per layer
(``SpectraGroup32QuantizedLayer``, spectra/engine.py:614-727) and dequantises
all of it at every step for the model's own attention.  Here the cache stays
in pages of 4-bit codes that sequences share out among themselves, the keys
enter it with the position rotation applied, and the attention reads the codes
(csrc/paged_kv.cu, csrc/paged_attn.cu, csrc/paged_prompt.cu):

    cache = PagedKVCache(num_pages, kv_heads, head_dim, page_size=64)
    batch = TokenBatch(block_tables, seq_lens)              # one new token per sequence
    batch = TokenBatch(block_tables, seq_lens, cu_q=cu_q, total=T, max_q=longest)   # ragged new tokens
    q = paged_kv_append(cache, batch, k, v, q=q, cos=cos, sin=sin)
    o = paged_attention(q, cache, batch)
    k_held, v_held = paged_kv_read(cache, batch)

A batch's arrays live on the device and are read by the kernels alone, so a
captured step can be replayed with other contents; ``max_len`` and ``max_q``
bound them.  There is no CPU path, and none is differentiable.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib as L
from . import _workspace as W

GROUP = 32
TILE_TOKENS = 16
HEAD_DIMS = (32, 64, 96, 128, 256)

_DT = {torch.float16: L.DT_F16, torch.bfloat16: L.DT_BF16}
_OUT_DT = {**_DT, torch.float32: L.DT_F32}


def tile_bytes(head_dim: int) -> int:
    """Bytes of one tile: 16 tokens of one head, keys and values (layout: include/spectra_b200.h)."""
    return 608 * (head_dim // GROUP)


class PagedKVCache:
    """Pages of one layer's INT4 keys and values: ``pool`` u8
    [num_pages, kv_heads, page_size / 16, tile_bytes], zeroed when made."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size < TILE_TOKENS or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from {TILE_TOKENS} to 65536, got {page_size}")
        pool = torch.zeros(num_pages, kv_heads, page_size // TILE_TOKENS, tile_bytes(head_dim), dtype=torch.uint8,
                           device=device)
        self._bind(pool, head_dim)

    @classmethod
    def from_pool(cls, pool: torch.Tensor, head_dim: int) -> "PagedKVCache":
        """A cache on an existing pool (pages may be apart: only the first stride is free)."""
        self = cls.__new__(cls)
        self._bind(pool, head_dim)
        return self

    def _bind(self, pool: torch.Tensor, head_dim: int) -> None:
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if pool.dtype != torch.uint8:
            raise TypeError(f"the pool must be uint8, got {pool.dtype}")
        if pool.dim() != 4 or pool.shape[3] != tile_bytes(head_dim):
            raise ValueError(f"the pool must be [num_pages, kv_heads, page_size / 16, {tile_bytes(head_dim)}], "
                             f"got {tuple(pool.shape)}")
        _, heads, tiles, tile = pool.shape
        if pool.numel() and (pool.stride(3) != 1 or (tiles > 1 and pool.stride(2) != tile)
                             or (heads > 1 and pool.stride(1) != tiles * tile)):
            raise ValueError("a page of the pool must be contiguous")
        if not pool.is_cuda:
            raise RuntimeError(f"spectra_b200.paged: the pool must be a CUDA tensor (no CPU path), got {pool.device}")
        self.pool, self.head_dim, self.kv_heads, self.page_size = pool, head_dim, heads, tiles * TILE_TOKENS
        self.num_pages, self._index = pool.shape[0], pool.get_device()
        stride = pool.stride(0) if self.num_pages > 1 else heads * tiles * tile
        self._c = L.PagedCache(pool.data_ptr(), stride, self.num_pages, heads, head_dim, self.page_size)
        self._at = ctypes.addressof(self._c)


class TokenBatch:
    """The sequences a step works on and their new tokens.

    ``block_tables`` int32 [B, width]: the pages of each sequence in order.
    ``seq_lens`` int32 [B]: tokens of each sequence, the new ones included
    (0: a slot that holds none).  The new tokens are a sequence's last ones;
    they are rows ``cu_q[b] .. cu_q[b + 1]`` of the token tensors (int32
    [B + 1]), or, without ``cu_q``, ``q_len`` rows each.  Host bounds:
    ``total`` rows, at most ``max_q`` of one sequence (the attention's results
    of rows past it are 0), ``max_len`` over seq_lens (default: what the tables
    can hold).
    """

    def __init__(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                 q_len: Optional[int] = None, total: Optional[int] = None, max_q: Optional[int] = None,
                 max_len: Optional[int] = None):
        for name, t in (("block_tables", block_tables), ("seq_lens", seq_lens), ("cu_q", cu_q)):
            if t is None:
                continue
            if t.dtype != torch.int32:
                raise TypeError(f"{name} must be int32, got {t.dtype}")
            if not t.is_cuda or t.device != block_tables.device:
                raise RuntimeError(f"spectra_b200.paged: {name} must be on the tables' CUDA device (no CPU path), got {t.device}")
        if block_tables.dim() != 2 or seq_lens.dim() != 1 or seq_lens.shape[0] != block_tables.shape[0]:
            raise ValueError(f"block_tables must be [B, width] and seq_lens [B], got {tuple(block_tables.shape)} and "
                             f"{tuple(seq_lens.shape)}")
        B, width = block_tables.shape
        if width > 1 and block_tables.stride(1) != 1:
            raise ValueError("block_tables must have unit stride along a sequence's pages")
        if B > 1 and seq_lens.stride(0) != 1:
            raise ValueError("seq_lens must be contiguous")
        if cu_q is None:
            q_len = 1 if q_len is None else int(q_len)
            total = B * q_len if total is None else int(total)
            max_q = q_len if max_q is None else int(max_q)
            if q_len < 0 or total != B * q_len or max_q < q_len:
                raise ValueError(f"{B} sequences of {q_len} new tokens each do not make total={total}, max_q={max_q}")
        else:
            if q_len is not None:
                raise ValueError("cu_q and q_len exclude each other")
            if cu_q.dim() != 1 or cu_q.shape[0] != B + 1 or (B and cu_q.stride(0) != 1):
                raise ValueError(f"cu_q must be contiguous [{B + 1}], got {tuple(cu_q.shape)}")
            if total is None or max_q is None:
                raise ValueError("cu_q needs total and max_q (host numbers: the kernels do not wait for the device)")
            total, max_q = int(total), int(max_q)
            if total < 0 or max_q < 0 or (total and not max_q):
                raise ValueError(f"total={total}, max_q={max_q}")
        if max_len is not None and max_len < 0:
            raise ValueError(f"max_len={max_len}")
        self.block_tables, self.seq_lens, self.cu_q = block_tables, seq_lens, cu_q
        self.batch, self.q_len, self.total, self.max_q, self.max_len = B, q_len, total, max_q, max_len
        self._index = block_tables.get_device()
        self._like: dict = {}
        self._c = L.TokenBatch(block_tables.data_ptr(), block_tables.stride(0) if B > 1 else width, width,
                               seq_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), B, q_len or 0, total,
                               max_q, 2**31 - 1 if max_len is None else int(max_len))
        self._at = ctypes.addressof(self._c)

    def _limit(self, cache: PagedKVCache) -> int:
        most = self.block_tables.shape[1] * cache.page_size
        return most if self.max_len is None else min(most, self.max_len)


def _rows(name: str, t: torch.Tensor, cache: PagedKVCache, batch: TokenBatch, heads: Optional[int]) -> torch.Tensor:
    """Checks a token tensor [total, heads, head_dim]; unit stride along a head."""
    if t.get_device() != cache._index:
        raise RuntimeError(f"spectra_b200.paged: {name} must be on the cache's CUDA device (no CPU path), got {t.device}")
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if t.dim() != 3 or t.shape[0] != batch.total or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [{batch.total}, {'heads' if heads is None else heads}, {cache.head_dim}], "
                         f"got {tuple(t.shape)}")
    return t if t.stride(2) == 1 else t.contiguous()


def _strided(name: str, t: torch.Tensor, cache: PagedKVCache, batch: TokenBatch, heads: Optional[int]):
    """The tensor with its token and head strides; the common case in few steps
    (a call's host time is what a single token waits for)."""
    ts, hs, unit = t.stride() if t.dim() == 3 else (0, 0, 0)
    if unit != 1 or t.get_device() != cache._index or t.dtype not in _DT or t.shape != (
            batch.total, t.shape[1] if heads is None else heads, cache.head_dim):
        t = _rows(name, t, cache, batch, heads)
        ts, hs, _ = t.stride()
    return t, ts, hs


def _other_device():
    raise RuntimeError("spectra_b200.paged: the batch's arrays must be on the cache's device")


_FNS: dict = {}  # the library's functions, looked up once


def _call(index: int, fn: str, *args) -> None:
    f = _FNS.get(fn)
    if f is None:
        f = _FNS[fn] = getattr(L.lib(), fn)
    if torch._C._cuda_getDevice() == index:
        st = f(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = f(*args, torch._C._cuda_getCurrentRawStream(index))
    if st:
        L.check(fn, st)


def paged_kv_append(cache: PagedKVCache, batch: TokenBatch, k: torch.Tensor, v: torch.Tensor,
                    q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                    sin: Optional[torch.Tensor] = None, interleaved: bool = False,
                    out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Append the batch's new tokens ``k``, ``v`` [total, kv_heads, D] to the
    cache, and return ``q`` [total, q_heads, D] rotated (None without q).

    ``cos``, ``sin`` fp32 [positions, rotary / 2]: the angles of each position;
    the first ``rotary`` features of q and k are turned (halves, or neighbours
    with ``interleaved``); without them nothing is turned.  All in fp32, the
    queries rounded once, the keys quantised without rounding in between.
    Groups that hold a NaN or infinity make their token's key NaN, so every row
    that looks at it is NaN and no other.  Token tensors may be views (any
    token and head strides), of a fused projection for example.  ``out``, for the
    rotated queries, shares no element with q, k or v."""
    index = cache._index
    if batch._index != index:
        _other_device()
    k, k_ts, k_hs = _strided("k", k, cache, batch, cache.kv_heads)
    v, v_ts, v_hs = _strided("v", v, cache, batch, cache.kv_heads)
    dt = k.dtype
    rotary = rows = cs = 0
    cp = sp = None
    if cos is not None or sin is not None:
        cos, sin, rotary, rows, cs = _angles(cos, sin, cache, batch, interleaved)
        if rotary:
            cp, sp = cos.data_ptr(), sin.data_ptr()
    qp = op = None
    heads = q_ts = q_hs = o_ts = o_hs = 0
    if q is not None:
        q, q_ts, q_hs = _strided("q", q, cache, batch, None)
        heads = q.shape[1]
        if out is None:
            out = torch.empty_like(q)
            o_ts, o_hs, unit = out.stride()
            if unit != 1:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                o_ts, o_hs, _ = out.stride()
        else:
            given, o_ts, o_hs = _strided("out", out, cache, batch, heads)
            if given is not out:
                raise ValueError("out must have unit stride along a head")
            _own_elements(out)
            if _overlap(out, q) or _overlap(out, k) or _overlap(out, v):
                raise ValueError("out must not overlap q, k or v")
        if q.dtype != dt or out.dtype != dt:
            raise TypeError("q, k, v and out must have one dtype")
        qp, op = q.data_ptr(), out.data_ptr()
    if v.dtype != dt:
        raise TypeError("q, k, v and out must have one dtype")
    _call(index, "spectra_paged_kv_append", cache._at, batch._at, _DT[dt], heads, qp, q_ts, q_hs, op, o_ts, o_hs,
          k.data_ptr(), k_ts, k_hs, v.data_ptr(), v_ts, v_hs, cp, sp, rows, cs, rotary, interleaved)
    return out if q is not None else None


def _angles(cos, sin, cache: PagedKVCache, batch: TokenBatch, interleaved: bool):
    if cos is None or sin is None:
        raise ValueError("cos and sin come together")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    if cos.get_device() != cache._index or sin.get_device() != cache._index:
        raise RuntimeError("spectra_b200.paged: cos and sin must be on the cache's CUDA device")
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError(f"cos and sin must be [positions, rotary / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    strides = cos.stride()
    if strides[1] != 1 or sin.stride() != strides:
        cos, sin = cos.contiguous(), sin.contiguous()
        strides = cos.stride()
    rows, half = cos.shape
    rotary = 2 * half
    if rotary > cache.head_dim or rotary % (8 if interleaved else 16):
        raise ValueError(f"the rotated part must be a multiple of {8 if interleaved else 16} and at most "
                         f"{cache.head_dim}, got {rotary}")
    if rows < batch._limit(cache):
        raise ValueError(f"cos and sin have {rows} positions, the batch may hold {batch._limit(cache)}")
    return cos, sin, rotary, rows, strides[0]


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + span * t.element_size()


def _runs(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """Where the tensor's runs of consecutive elements start (addresses in order), and their bytes."""
    (T, H, D), (ts, hs, _), size = t.shape, t.stride(), t.element_size()
    if hs == D or H == 1:
        return t.data_ptr() + torch.arange(T if ts else 1) * (ts * size), H * D * size
    starts = torch.arange(T if ts else 1)[:, None] * ts + torch.arange(H) * hs
    return t.data_ptr() + torch.unique(starts) * size, D * size


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether [tokens, heads, D] tensors of unit stride along a head share an element.  Views of one
    buffer that lie between each other's rows do not."""
    lo, hi = _extent(a)
    blo, bhi = _extent(b)
    if lo >= bhi or blo >= hi:
        return False
    (sa, la), (sb, lb) = _runs(a), _runs(b)
    i = torch.searchsorted(sa, sb, right=True)  # the first run of a that starts past b's; one of either side touches it
    first = torch.cat([sb[:1] - la, sa])[i]
    after = torch.cat([sa, sb[-1:] + lb])[i]
    return bool((first + la > sb).any() or (sb + lb > after).any())


def _own_elements(out: torch.Tensor) -> None:
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError("out must not be an expanded tensor")


def paged_kv_read(cache: PagedKVCache, batch: TokenBatch, dtype: torch.dtype = torch.bfloat16):
    """Keys and values [total, kv_heads, D] that the cache holds of the batch's
    new tokens: ``(q - z) * s`` rounded once to ``dtype`` (exact in fp32); 0 for
    padding.  ``cu_q`` of cumulated seq_lens reads whole sequences."""
    if batch._index != cache._index:
        _other_device()
    if dtype not in _OUT_DT:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    like = batch._like.get((dtype, cache.kv_heads, cache.head_dim))
    if like is None:  # a shape to allocate by, without memory of its own
        like = torch.empty(1, 1, 1, dtype=dtype, device=cache.pool.device).expand(batch.total, cache.kv_heads, cache.head_dim)
        batch._like[dtype, cache.kv_heads, cache.head_dim] = like
    k = torch.empty_like(like, memory_format=torch.contiguous_format)
    v = torch.empty_like(like, memory_format=torch.contiguous_format)
    _call(cache._index, "spectra_paged_kv_read", cache._at, batch._at, k.data_ptr(), v.data_ptr(), _OUT_DT[dtype])
    return k, v


# Partial results of split sequences, one buffer per (device, stream, head_dim),
# kept for the process: calls on one stream never overlap.  Zeroed once; every
# call leaves its counters zero.  The size does not depend on the batch, so a
# buffer is never replaced and a captured graph's address stays good.  A capture
# on a stream that has none gets its own (_workspace.py).
_WORKSPACES: dict = {}


def _workspace(index: int, head_dim: int) -> Tuple[int, int]:
    stream = torch._C._cuda_getCurrentRawStream(index)
    key = (index, stream, head_dim)
    ws = _WORKSPACES.get(key)
    if ws is None:
        nbytes, dev = L.lib().spectra_paged_attention_workspace_bytes(head_dim), torch.device("cuda", index)
        buf = W.captured(dev, stream, ("paged", head_dim), nbytes, L.PAGED_COUNTER_BYTES)
        if buf is not None:
            return buf.data_ptr(), nbytes
        buf = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
        ws = _WORKSPACES[key] = (buf.data_ptr(), nbytes, buf)
    return ws[0], ws[1]


def paged_attention(q: torch.Tensor, cache: PagedKVCache, batch: TokenBatch, *, scale: Optional[float] = None,
                    causal: bool = True, window: int = 0, softcap: float = 0.0,
                    alibi_slopes: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the batch's new tokens ``q`` [total, q_heads, D] over the
    cache (append them first); the result has q's shape and dtype.

    Row (position p, head h) sees the keys n < seq_len with ``causal`` n <= p,
    with ``window`` > 0 n > p - window; its scores are ``scale`` (default
    1 / sqrt(D)) times the products, then ``softcap * tanh(score / softcap)``,
    then plus ``alibi_slopes[h] * (n - p)`` (fp32 [q_heads]).  q_heads is a
    multiple of kv_heads; consecutive heads share one.  A row that sees no key
    is 0.  Scores, softmax statistics and sums are fp32.  ``out`` may be q
    itself (the same strides); otherwise they share no element.

    Partial results lie in a workspace of the current stream (17 MB for heads of
    128, kept for the process).  A graph captured on a stream that has called
    this before holds that stream's: do not let its replays overlap other calls
    of that stream, or replays of another graph captured there.  Captured on a
    stream that has not, it holds its own."""
    index = cache._index
    if batch._index != index:
        _other_device()
    q, q_ts, q_hs = _strided("q", q, cache, batch, None)
    heads = q.shape[1]
    if heads % cache.kv_heads or not heads:
        raise ValueError(f"q has {heads} heads, not a multiple of the cache's {cache.kv_heads}")
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf or not 0.0 <= softcap < math.inf:
        raise ValueError(f"scale must be positive and softcap not negative (both finite), got {scale} and {softcap}")
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    slopes = None
    if alibi_slopes is not None:
        if alibi_slopes.dtype != torch.float32 or alibi_slopes.shape != (heads,):
            raise ValueError(f"alibi_slopes must be float32 [{heads}]")
        if alibi_slopes.get_device() != index:
            raise RuntimeError("spectra_b200.paged: alibi_slopes must be on the cache's CUDA device")
        slopes = alibi_slopes if heads == 1 or alibi_slopes.stride(0) == 1 else alibi_slopes.contiguous()
    if out is None:
        out = torch.empty_like(q)
        o_ts, o_hs, unit = out.stride()
        if unit != 1:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            o_ts, o_hs, _ = out.stride()
    else:
        given, o_ts, o_hs = _strided("out", out, cache, batch, heads)
        if given is not out or out.dtype != q.dtype:
            raise ValueError("out must have q's dtype and unit stride along a head")
        _own_elements(out)
        if (out.data_ptr() != q.data_ptr() or o_ts != q_ts or o_hs != q_hs) and _overlap(out, q):
            raise ValueError("out must not overlap q, unless it is q")
    ws, nbytes = _workspace(index, cache.head_dim)
    _call(index, "spectra_paged_attention", cache._at, batch._at, _DT[q.dtype], heads, q.data_ptr(), q_ts, q_hs,
          out.data_ptr(), o_ts, o_hs, scale, softcap, None if slopes is None else slopes.data_ptr(), causal,
          min(window, 2**31 - 1), ws, nbytes)
    return out
