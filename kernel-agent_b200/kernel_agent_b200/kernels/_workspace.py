"""Scratch buffers of the kernels that leave counters at zero after every launch."""

from __future__ import annotations

import torch

_BUFFERS: dict[tuple, torch.Tensor] = {}


def workspace(op: str, device: torch.device, stream: int, nbytes: int, zero_bytes: int) -> torch.Tensor:
    """``nbytes`` of scratch for ``op`` on ``stream`` whose first ``zero_bytes`` are zero. The
    kernels put their counters there and leave them at zero, so a buffer is zeroed only when it
    is made, on the stream that uses it; ``op`` names everything that decides where the counters
    lie. While a CUDA graph is captured every call makes its own (it belongs to the graph, which
    zeroes it at every replay)."""
    if torch.cuda.is_current_stream_capturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:zero_bytes].zero_()
        return buf
    key = (op, device.index, stream, zero_bytes)
    buf = _BUFFERS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:zero_bytes].zero_()
        _BUFFERS[key] = buf
    return buf
