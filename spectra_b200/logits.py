"""Rules on a step's logits: penalties for repeated tokens, biases, a mask of
the tokens that may follow, and the greedy choice under them (csrc/logits.cu).

The reference's engine applies its penalties in torch between the head and
sample_token (spectra/engine.py:1626-1713); here one kernel does it in one pass:

    rules = LogitRules(ids=ids, lengths=lengths, prompt_lengths=prompts, repetition=1.1, allowed=grammar_bits)
    logits, tokens = adjust_logits(logits, rules, with_tokens=True)
    tokens = kernels.argmax(logits, rules=rules)            # the choice alone: no logits are written

The rules' tensors stay on the device and are read by the kernel alone, so a
captured step can be replayed with other contents.  There is no CPU path, and
nothing here is differentiable.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib as L

_DT = {torch.float16: L.DT_F16, torch.bfloat16: L.DT_BF16, torch.float32: L.DT_F32}


class LogitRules:
    """The rules of a batch of rows, one row per row of the logits (65535 at most).

    ``ids`` int32 [rows, most]: the tokens that each sequence holds, its prompt
    first; the first ``lengths`` int32 [rows] of them count (default: all), the
    first ``prompt_lengths`` int32 [rows] of those are the prompt (default:
    none).  ``repetition``, ``frequency``, ``presence``: a number, or fp32 [rows].
    ``bias_ids`` int32 and ``bias`` fp32 [rows, n]: added to the logits of those
    tokens; of an id that a row lists more than once the last one counts.
    ``allowed`` int32 [rows, words]: bit ``i % 32`` of word ``i // 32`` set where
    token i may follow.  A negative id names no token, so rows may be padded
    with -1.  Ids are the vocabulary's, also for a slice of it.

    A logit x of token v becomes, in fp32 and in this order:
      v among the ids:                  x / repetition if x > 0 else x * repetition
      v n > 0 times after the prompt:   x - frequency * n, then x - presence
      then x + bias; then -infinity where v is not allowed, whatever x was.
    """

    def __init__(self, ids: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                 prompt_lengths: Optional[torch.Tensor] = None,
                 repetition: Union[None, float, torch.Tensor] = None, frequency: Union[None, float, torch.Tensor] = None,
                 presence: Union[None, float, torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None):
        if (bias_ids is None) != (bias is None):
            raise ValueError("bias_ids and bias come together")
        if ids is None and any(x is not None for x in (lengths, prompt_lengths, repetition, frequency, presence)):
            raise ValueError("lengths and penalties need ids")
        wide = {"ids": ids, "bias_ids": bias_ids, "bias": bias, "allowed": allowed}
        some = next((t for t in wide.values() if t is not None), None)
        if some is None:
            raise ValueError("no rules: give ids, bias_ids and bias, or allowed")
        self.device, self.rows = some.device, some.shape[0] if some.dim() else -1
        if self.rows > 65535:
            raise ValueError(f"at most 65535 rows, got {self.rows}")
        for name, t in wide.items():
            if t is None:
                continue
            self._check(name, t, torch.float32 if name == "bias" else torch.int32)
            if t.dim() != 2 or t.shape[0] != self.rows:
                raise ValueError(f"{name} must be [{self.rows if self.rows >= 0 else 'rows'}, n], got {tuple(t.shape)}")
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError(f"{name} must have unit stride along a row")
        if bias is not None and bias.shape != bias_ids.shape:
            raise ValueError(f"bias_ids and bias must have one shape, got {tuple(bias_ids.shape)} and {tuple(bias.shape)}")
        if ids is not None and ids.shape[1] > L.MAX_RULE_IDS:
            raise ValueError(f"at most {L.MAX_RULE_IDS} ids a row, got {ids.shape[1]}")
        if bias is not None and bias.shape[1] > L.MAX_RULE_BIASES:
            raise ValueError(f"at most {L.MAX_RULE_BIASES} biases a row, got {bias.shape[1]}")
        if repetition is not None and not isinstance(repetition, torch.Tensor) and not repetition > 0:
            raise ValueError(f"repetition must be positive, got {repetition}")
        row = {}
        for name, t in (("lengths", lengths), ("prompt_lengths", prompt_lengths), ("repetition", repetition),
                        ("frequency", frequency), ("presence", presence)):
            if t is not None and not isinstance(t, torch.Tensor):
                if "lengths" in name:
                    raise TypeError(f"{name} must be an int32 tensor")
                t = torch.full((self.rows,), float(t), dtype=torch.float32, device=self.device)
            if t is not None:
                self._check(name, t, torch.int32 if "lengths" in name else torch.float32)
                if t.shape != (self.rows,) or (self.rows > 1 and t.stride(0) != 1):
                    raise ValueError(f"{name} must be contiguous [{self.rows}], got {tuple(t.shape)}")
            row[name] = t
        self._keep = (wide, row)
        self.words = 0 if allowed is None else allowed.shape[1]
        self._index, self._masked = some.get_device(), allowed is not None
        self._bytes: dict = {}  # of workspace, by what is asked for
        self._like = torch.empty(1, dtype=torch.int64, device=self.device).expand(self.rows)  # a shape to allocate by
        at = lambda t: None if t is None or not t.numel() else t.data_ptr()  # noqa: E731
        step = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
        self._c = L.LogitRules(
            at(ids), step(ids), 0 if ids is None else ids.shape[1], at(row["lengths"]), at(row["prompt_lengths"]),
            at(row["repetition"]), at(row["frequency"]), at(row["presence"]), at(bias_ids), step(bias_ids), at(bias),
            step(bias), 0 if bias is None else bias.shape[1], None if allowed is None else allowed.data_ptr(), step(allowed),
            self.words)
        self._at = ctypes.addressof(self._c)

    def _check(self, name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {str(dtype)[6:]}, got {t.dtype}")
        if not t.is_cuda or t.device != self.device:
            raise RuntimeError(f"spectra_b200.logits: the rules must be on one CUDA device (no CPU path), got {name} on {t.device}")


_FN = None  # the library's function, looked up once


def _apply(x: torch.Tensor, rules: LogitRules, idx_offset: int, out: Optional[torch.Tensor], idx, val) -> None:
    """x, out [M, N] of unit stride along a row; idx int64, val fp32 [M] (each optional)."""
    global _FN
    M, N = x.shape
    index = rules._index
    if x.get_device() != index:
        raise RuntimeError(f"spectra_b200.logits: the logits must be on the rules' CUDA device (no CPU path), got {x.device}")
    dt = _DT.get(x.dtype)
    if dt is None:
        raise TypeError(f"logits must be bf16, fp16 or fp32, got {x.dtype}")
    if M != rules.rows or N < 1:
        raise ValueError(f"the rules are of {rules.rows} rows, the logits {tuple(x.shape)}")
    if idx_offset < 0 or idx_offset + N > 2**31 - 65:
        raise ValueError(f"idx_offset={idx_offset} and {N} logits pass 32 bits")
    if rules.words * 32 < idx_offset + N and rules._masked:
        raise ValueError(f"allowed has {rules.words} words a row, {-(-(idx_offset + N) // 32)} are needed")
    if M == 0:
        return
    if _FN is None:
        _FN = L.lib().spectra_adjust_logits
    ws, nbytes = None, rules._bytes.get((N, dt, idx is None))
    if nbytes is None:
        nbytes = L.lib().spectra_adjust_logits_workspace_bytes(rules._at, M, N, dt, idx is not None)
        rules._bytes[N, dt, idx is None] = nbytes
    if nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        ws = buf.data_ptr()
    args = (rules._at, x.data_ptr(), dt, x.stride(0) if M > 1 else N, M, N, idx_offset,
            None if out is None else out.data_ptr(), 0 if out is None else _DT[out.dtype],
            0 if out is None else (out.stride(0) if M > 1 else N), None if idx is None else idx.data_ptr(),
            None if val is None else val.data_ptr(), ws, nbytes)
    if torch._C._cuda_getDevice() == index:
        st = _FN(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = _FN(*args, torch._C._cuda_getCurrentRawStream(index))
    if st:
        L.check("spectra_adjust_logits", st)


def _rows(logits: torch.Tensor) -> torch.Tensor:
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    step, unit = x.stride()
    return x if unit == 1 and (step >= x.shape[1] or x.shape[0] < 2) else x.contiguous()


def adjust_logits(logits: torch.Tensor, rules: LogitRules, *, out: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None, idx_offset: int = 0,
                  with_tokens: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``logits`` [..., N] under the rules, rounded once to ``out_dtype`` (default:
    theirs); column n is token ``n + idx_offset`` (a slice of the vocabulary).
    With ``with_tokens`` also the greedy choice, int64 [...]: idx_offset + the
    first column of the maximum among the allowed tokens, taken before the
    rounding (a NaN counts as the maximum), -1 where no token is allowed.

    ``out`` [..., N], unit stride along a row, may be the logits themselves;
    otherwise they share no element."""
    shape = logits.shape
    flat = len(shape) == 2
    if not shape or shape[-1] < 1:
        raise ValueError(f"logits must be [..., N], got {tuple(shape)}")
    x = _rows(logits)
    if out is None:
        if out_dtype is None or out_dtype == x.dtype:
            y = torch.empty_like(x, memory_format=torch.contiguous_format)
        elif out_dtype in _DT:
            y = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
        else:
            raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
        res = y if flat else y.reshape(shape)
    else:
        if out.shape != shape or out.device != logits.device or (out_dtype or out.dtype) != out.dtype:
            raise ValueError(f"out must be {tuple(shape)} on the logits' device, of out_dtype where that is given")
        if out.dtype not in _DT:
            raise TypeError(f"out must be bf16, fp16 or fp32, got {out.dtype}")
        y = out if flat else out.view(-1, shape[-1])
        if (y.shape[1] > 1 and y.stride(1) != 1) or (y.shape[0] > 1 and y.stride(0) < y.shape[1]):
            raise ValueError("out must have unit stride along a row, and rows that do not overlap")
        same = y.data_ptr() == x.data_ptr() and y.dtype == x.dtype and (y.shape[0] < 2 or y.stride(0) == x.stride(0))
        if not same and _overlap(x, y):
            raise ValueError("out must not overlap the logits, unless it is the logits")
        res = out
    if not with_tokens:
        _apply(x, rules, idx_offset, y, None, None)
        return res
    idx = torch.empty_like(rules._like, memory_format=torch.contiguous_format)
    _apply(x, rules, idx_offset, y, idx, None)
    return res, idx if flat else idx.reshape(shape[:-1])


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether [M, N] tensors of unit stride along a row may share an element (by their rows' extents)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()

    if not x.numel():
        return False
    (a, b), (c, d) = span(x), span(y)
    if a >= d or c >= b:
        return False
    rs = x.stride(0) * x.element_size()
    if x.shape[0] > 1 and y.stride(0) * y.element_size() == rs:  # rows of one pitch: columns beside each other?
        gap, wx, wy = (c - a) % rs, x.shape[1] * x.element_size(), y.shape[1] * y.element_size()
        return gap < wx or gap + wy > rs
    return True
