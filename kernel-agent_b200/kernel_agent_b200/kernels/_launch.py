"""What a launch needs from torch, at a decode step's pace: the tensors' device, the current
stream as the C ABI takes it, a device guard only where one is needed, and scratch buffers of the
kernels that leave counters at zero after every launch."""

from __future__ import annotations

from contextlib import nullcontext

import torch

from .. import _native as nat

_BUFFERS: dict[tuple, torch.Tensor] = {}
_NO_GUARD = nullcontext()


def device_of(*tensors: torch.Tensor | None) -> int:
    """The index of the CUDA device that all given tensors are on (the checks and errors of
    :func:`kernel_agent_b200._native.require_cuda`)."""
    dev = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device() if isinstance(t, torch.Tensor) else -1
        if at < 0 or (dev >= 0 and at != dev):
            break
        dev = at
    else:
        if dev in nat._checked_devices:
            return dev
    found = nat.require_cuda(*tensors)
    return torch.cuda.current_device() if found.index is None else found.index


def guard(device: int):
    """A context in which ``device`` is the current one."""
    return _NO_GUARD if torch._C._cuda_getDevice() == device else torch.cuda.device(device)


def stream_of(device: int) -> int:
    """The current CUDA stream of ``device``, as the void* the ABI takes."""
    return torch._C._cuda_getCurrentRawStream(device)


def workspace(op: tuple | str, device: int, stream: int, nbytes: int, zero_bytes: int) -> torch.Tensor:
    """``nbytes`` of scratch for ``op`` on ``stream`` whose first ``zero_bytes`` are zero. The
    kernels put their counters there and leave them at zero, so a buffer is zeroed only when it
    is made, on the stream that uses it; ``op`` names everything that decides where the counters
    lie. While a CUDA graph is captured every call makes its own (it belongs to the graph, which
    zeroes it at every replay)."""
    if torch._C._cuda_isCurrentStreamCapturing():
        return _make(device, nbytes, zero_bytes)
    key = (op, device, stream, zero_bytes)
    buf = _BUFFERS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _BUFFERS[key] = _make(device, nbytes, zero_bytes)
    return buf


def _make(device: int, nbytes: int, zero_bytes: int) -> torch.Tensor:
    buf = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
    if zero_bytes:
        buf[:zero_bytes].zero_()
    return buf
