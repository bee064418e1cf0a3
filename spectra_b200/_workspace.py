"""Workspaces of calls that are being captured in a CUDA graph.

A call's workspace is made once per stream, zeroed, and kept.  While the
stream is being captured that would go wrong: the zeroing would become a node
of this one graph and the memory would come from its pool, yet every later
call on the stream would take the buffer for a zeroed one, before the graph's
first replay or after its end.  So a captured call that finds no kept buffer
gets one that belongs to the capture: the graph zeroes it at every replay, and
no call outside it ever sees it.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

# Buffers of the newest capture: {capture id: {key: buffer}}.  Dropped with the
# next capture; until the graph itself is gone its pool keeps the memory.
_CAPTURED: dict = {}


def captured(device: torch.device, stream: int, key, nbytes: int, zeroed: int) -> Optional[torch.Tensor]:
    """The buffer ``key`` of the capture that ``stream`` is part of, at least
    ``nbytes`` long and zero in its first ``zeroed`` when the graph reaches this
    call for the first time; None if the stream is not being captured."""
    capture = L.lib().spectra_stream_capture_id(stream)
    if not capture:
        return None
    bufs = _CAPTURED.get(capture)
    if bufs is None:
        _CAPTURED.clear()
        bufs = _CAPTURED[capture] = {}
    key = (device.index, stream, key)
    buf = bufs.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:zeroed].zero_()
        bufs[key] = buf
    return buf
