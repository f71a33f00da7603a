"""What a launch needs from torch, at a decode step's pace: the tensors' device, the current
stream as the C ABI takes it, a device guard only where one is needed, and scratch buffers."""

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


def workspace(op: str, device: int, stream: int, nbytes: int) -> torch.Tensor:
    """``nbytes`` of scratch for ``op`` on ``stream``, kept for its next call there (a call's contents
    mean nothing to the next). While a CUDA graph is captured every call makes its own: it belongs to
    the graph, which may be replayed beside other work."""
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
    key = (op, device, stream)
    buf = _BUFFERS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _BUFFERS[key] = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
    return buf


def to_device(values: list, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A small host list as a device tensor, without waiting for the GPU (through pinned memory)."""
    return torch.tensor(values, dtype=dtype).pin_memory().to(device, non_blocking=True)
