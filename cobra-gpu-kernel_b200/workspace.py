"""The workspace of a module: grown on demand, kept where a caller's graph needs it."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


class HoldsWorkspace:
    """``_ws_bytes`` bytes from ``workspace_ptr`` on (1024-byte aligned, status block
    first). A workspace that a call outgrows is replaced; if it was current during a
    stream capture it is kept as long as the module is, for a caller's graph goes on
    using it."""

    _ws: Optional[torch.Tensor] = None
    _ws_off = 0
    _ws_bytes = 0
    _ws_captured = False
    _ws_kept: Tuple[Tuple[torch.Tensor, int], ...] = ()

    @property
    def workspace_ptr(self) -> int:
        return self._ws.data_ptr() + self._ws_off

    def _hold_workspace(self, need: int, device: torch.device) -> bool:
        """Hold ``need`` bytes on ``device`` at least; whether the workspace is a new one."""
        capturing = torch.cuda.is_current_stream_capturing()
        if self._ws is not None and self._ws.device == device and self._ws_bytes >= need:
            self._ws_captured |= capturing
            return False
        if self._ws_captured:
            self._ws_kept += ((self._ws, self._ws_off),)
        self._ws, self._ws_captured = None, False
        buf = torch.empty(need + 1024, dtype=torch.uint8, device=device)
        self._ws, self._ws_off, self._ws_bytes = buf, (-buf.data_ptr()) % 1024, need
        self._ws_captured = capturing
        with torch.cuda.device(device):
            _lib.check(_lib.lib().b200l_clear_status(self.workspace_ptr, torch.cuda.current_stream(device).cuda_stream))
        return True

    def check_status(self) -> None:
        """Synchronise and raise if a kernel recorded a device-side failure."""
        held = self._ws_kept if self._ws is None else (*self._ws_kept, (self._ws, self._ws_off))
        for buf, off in held:
            with torch.cuda.device(buf.device):
                rc = _lib.lib().b200l_read_status(buf.data_ptr() + off, torch.cuda.current_stream(buf.device).cuda_stream)
            _lib.check(rc)
