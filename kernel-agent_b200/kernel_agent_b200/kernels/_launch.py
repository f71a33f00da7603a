"""What a launch needs from torch, at a decode step's pace: the tensors' device, the current
stream as the C ABI takes it, calls with that device current, and scratch buffers."""

from __future__ import annotations

import torch

from .. import _native as nat

_ENTRIES: dict[str, object] = {}


def device_of(*tensors: torch.Tensor | None) -> int:
    """The index of the CUDA device that all given tensors are on (the checks and errors of
    :func:`kernel_agent_b200._native.require_cuda`)."""
    try:
        dev = tensors[0].get_device()
        for t in tensors:
            if t is not None and t.get_device() != dev:
                break
        else:
            if dev in nat._checked_devices:
                return dev
    except AttributeError:
        pass  # not a tensor: refused below
    found = nat.require_cuda(*tensors)
    return torch.cuda.current_device() if found.index is None else found.index


def call(name: str, device: int, *args) -> None:
    """Entry point ``name`` with ``device`` current; a non-zero status raises as in
    :func:`kernel_agent_b200._native.call`."""
    entry = _ENTRIES.get(name)
    if entry is None:
        entry = _ENTRIES[name] = getattr(nat.load(), name)
    if torch._C._cuda_getDevice() == device:
        status = entry(*args)
    else:
        with torch.cuda.device(device):
            status = entry(*args)
    if status:
        nat.refuse(name, status)


def stream_of(device: int) -> int:
    """The current CUDA stream of ``device``, as the void* the ABI takes."""
    return torch._C._cuda_getCurrentRawStream(device)


def workspace(device: int, nbytes: int) -> torch.Tensor:
    """``nbytes`` of scratch for one call on the current stream. Each call takes its own from the
    allocator: a call passes data from launch to launch through it, and another thread's call on the
    same stream may enqueue its launches between them. The caller holds it until its launches are
    enqueued; the allocator then gives it to later work of this stream only."""
    return torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))


def keep(table: dict, key: tuple, value):
    """``table[key] = value``, the table emptied first where it holds 1024 layouts: enough for a program's
    steps, and bounded where shapes change without end. Returns ``value``."""
    if len(table) >= 1024:
        table.clear()
    table[key] = value
    return value


def to_device(values: list, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A small host list as a device tensor, without waiting for the GPU (through pinned memory)."""
    return torch.tensor(values, dtype=dtype).pin_memory().to(device, non_blocking=True)
