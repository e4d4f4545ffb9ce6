"""Workspaces: where their memory comes from, and the one that a module holds."""

from __future__ import annotations

import contextlib
import ctypes
from typing import Iterator, Optional, Tuple

import torch

from . import _lib


def _cleared(need: int, device: torch.device) -> Tuple[torch.Tensor, int]:
    buf = torch.empty(need + 1024, dtype=torch.uint8, device=device)
    off = (-buf.data_ptr()) % 1024
    _lib.check(_lib.lib().b200l_clear_status(buf.data_ptr() + off, torch.cuda.current_stream(device).cuda_stream))
    return buf, off


@contextlib.contextmanager
def _beside_the_capture(device: torch.device) -> Iterator[torch.cuda.Stream]:
    """A stream that is not being captured, current, in a thread that may allocate and
    wait on it although another is."""
    mode = ctypes.c_int32(_lib.CAPTURE_RELAXED)
    _lib.check(_lib.lib().b200l_exchange_capture_mode(ctypes.byref(mode)))
    try:
        for _ in range(64):                     # (torch hands out the same 32 streams in turn)
            stream = torch.cuda.Stream(device)
            with torch.cuda.stream(stream):
                if not torch.cuda.is_current_stream_capturing():
                    break
        else:
            raise RuntimeError("every stream is being captured: run the step once before its capture")
        with torch.cuda.stream(stream):
            yield stream
    finally:
        _lib.check(_lib.lib().b200l_exchange_capture_mode(ctypes.byref(mode)))


def new_workspace(need: int, device: torch.device) -> Tuple[torch.Tensor, int]:
    """(tensor, byte in it) of a workspace of ``need`` bytes at a 1024-byte boundary, its
    status block cleared in the order of ``device``'s current stream.

    While that stream is captured nothing of this goes into the graph: a second graph
    may be replayed before the first, and a status block that every step clears tells
    nothing of the step before. The memory comes from another stream, and so not from
    the graph's pool, where what the graph did earlier would be done to it again by each
    replay; and it is cleared on the spot."""
    with torch.cuda.device(device):
        if not torch.cuda.is_current_stream_capturing():
            return _cleared(need, device)
        with _beside_the_capture(device) as stream:
            made = _cleared(need, device)
            stream.synchronize()
        return made


class HoldsWorkspace:
    """``_ws_bytes`` bytes from ``workspace_ptr`` on (1024-byte aligned, status block
    first). A workspace that a call outgrows is replaced; if it was current during a
    stream capture it is kept as long as the module is, for a caller's graph goes on
    using it."""

    _ws: Optional[torch.Tensor] = None
    _ws_off = 0
    _ws_bytes = 0
    _ws_captured = False           # a capture used it
    _ws_aside = False              # a capture made it, on another stream
    _ws_kept: Tuple[Tuple[torch.Tensor, int], ...] = ()

    @property
    def workspace_ptr(self) -> int:
        return self._ws.data_ptr() + self._ws_off

    def _hold_workspace(self, need: int, device: torch.device) -> bool:
        """Hold ``need`` bytes on ``device`` at least; whether the workspace is a new one."""
        capturing = torch.cuda.is_current_stream_capturing()
        if self._ws is not None and self._ws.device == device and self._ws_bytes >= need:
            self._ws_captured |= capturing
            if self._ws_aside and not capturing:
                self._ws.record_stream(torch.cuda.current_stream(device))
            return False
        if self._ws_captured:
            self._ws_kept += ((self._ws, self._ws_off),)
        self._ws, self._ws_captured = None, False
        (self._ws, self._ws_off), self._ws_bytes = new_workspace(need, device), need
        self._ws_captured = self._ws_aside = capturing
        return True

    def check_status(self) -> None:
        """Synchronise and raise if a kernel recorded a device-side failure."""
        held = self._ws_kept if self._ws is None else (*self._ws_kept, (self._ws, self._ws_off))
        for buf, off in held:
            with torch.cuda.device(buf.device):
                rc = _lib.lib().b200l_read_status(buf.data_ptr() + off, torch.cuda.current_stream(buf.device).cuda_stream)
            _lib.check(rc)
