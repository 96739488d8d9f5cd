"""Device scratch that a kernel's calls share, also under CUDA graph capture.

The kernels keep ticket words at the start of their scratch that have to be
zero when a call begins and are zero again when it ends. Eager calls of one
stream run one after another and share a buffer, which may be replaced by a
larger one at any time. A captured call is replayed later, next to whatever
runs then, so it never takes the eager buffer: every capture has a buffer of
its own from the graph's memory pool, and the fill of its ticket words is
recorded in the graph ahead of the first call that takes it.
"""
from __future__ import annotations

import torch

from ._lib import lib


class Scratch:
    """Buffers by stream, and by stream and capture. ``head``: bytes at the
    start that a call needs zeroed (0: all)."""

    def __init__(self, head: int = 0):
        self.head = head
        self._eager: dict = {}
        self._capture = 0          # the capture that the buffers below belong to
        self._captured: dict = {}

    def get(self, nbytes: int, device, st: int) -> torch.Tensor:
        """At least ``nbytes`` for a call on ``st``, the current stream."""
        # (the default stream, handle 0, cannot be captured)
        if st and torch.cuda.is_current_stream_capturing():
            capture = lib.vb_stream_capture_id(st)
            if not capture or capture != self._capture:
                self._captured.clear()
                self._capture = capture
            buf = self._captured.get((device, st))
            if buf is None or buf.numel() < nbytes:
                buf = torch.empty(max(nbytes, self.head), dtype=torch.uint8, device=device)
                buf[:self.head or nbytes].zero_()
                self._captured[device, st] = buf
            return buf
        if self._captured:  # the graphs' pools keep them now
            self._captured.clear()
        buf = self._eager.get((device, st))
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, self.head), dtype=torch.uint8, device=device)
            self._eager[device, st] = buf
        return buf


__all__ = ["Scratch"]
