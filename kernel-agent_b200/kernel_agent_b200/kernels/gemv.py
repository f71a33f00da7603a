"""Weight-only FP4 linear for the few tokens of a decode step.

:func:`fp4_w4a16_linear` multiplies activations as they are (no quantisation of ``x``) with a
weight that :func:`kernel_agent_b200.kernels.quant.quantize_fp4` made, in the layout that
:func:`~kernel_agent_b200.kernels.quant.fp4_w4a4_linear` reads: one copy of a weight serves the
prompt (W4A4 on the tensor cores' FP4 rate) and the single tokens, where only the weight's bytes
count. The reference's decode example for such weights is
``src/kernel_agent/agent/examples/cuda_fp4_gemv.py``.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _native as nat
from . import quant as q
from ._launch import call, device_of, keep, stream_of, workspace
from .gemm import _bias

_FORMATS = {"nvfp4": (nat.KAB_NVFP4, 16, torch.float8_e4m3fn), "mxfp4": (nat.KAB_MXFP4, 32, torch.float8_e8m0fnu)}
_PLANS: dict[tuple, int] = {}


def _plan(m: int, n: int, k: int, fmt: int, dtype: int, device: int) -> int:
    """Workspace bytes of a shape (asked once)."""
    key = (m, n, k, fmt, dtype, device)
    nbytes = _PLANS.get(key)
    if nbytes is None:
        found = ctypes.c_size_t(0)
        call("kab_gemv_fp4_workspace", device, m, n, k, fmt, dtype, ctypes.byref(found))
        nbytes = keep(_PLANS, key, int(found.value))
    return nbytes


def fp4_w4a16_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, tensor_scale: torch.Tensor | float,
                     bias: torch.Tensor | None = None, *, fmt: str = "nvfp4") -> torch.Tensor:
    """``x @ Wᵀ (+ bias)`` with ``W = e2m1(codes) * scales * tensor_scale``: products of ``x`` and the
    weight's values, fp32 sums, ``acc * tensor_scale (+ bias)`` and one rounding to ``x``'s dtype. The
    products are exact for bf16 and fp16 ``x`` down to 2^-28 of a row's largest finite value; fp32 ``x``
    enters with 22 bits (the result's error is about 3e-7 of its size).

    ``x [..., K]``; ``codes [N, K / 2]`` (packed e2m1, low nibble first); ``scales [N, K /
    block]`` (e4m3 per 16 for ``fmt="nvfp4"``, e8m0 per 32 for ``"mxfp4"``) or the same already
    swizzled (flat, 128 x 4 blocks); ``tensor_scale`` one value or one per row of the weight.
    Made for up to about 32 rows of ``x``, where the weight's bytes bound it; more rows work, the
    weight being read again for every 32. Against :func:`~kernel_agent_b200.kernels.quant.fp4_w4a4_linear`
    on the same codes and scales: 29.6 us and 103 for one row of 28672 x 8192 NVFP4, 94 and 99 for 32;
    MXFP4 29.5 and 79 for one row, 74 and 77 for 16, 120 and 72 for 32. So from about 32 rows of NVFP4
    and 20 of MXFP4 that one is the faster, where ``x`` may be rounded to FP4."""
    if fmt not in _FORMATS:
        raise ValueError(f"unknown FP4 format {fmt!r} (one of {', '.join(_FORMATS)})")
    code, block, kind = _FORMATS[fmt]
    device = device_of(x, codes, scales, bias)
    if x.dim() < 1 or codes.dim() != 2:
        raise ValueError(f"expected x [..., K] and codes [N, K / 2]; got {tuple(x.shape)}, {tuple(codes.shape)}")
    n, half = codes.shape
    k = x.shape[-1]
    if k % block:
        raise ValueError(f"the last dimension {k} is not a multiple of the {fmt} block ({block})")
    if half * 2 != k or codes.element_size() != 1:
        raise ValueError(f"codes {tuple(codes.shape)} {codes.dtype} do not fit x {tuple(x.shape)}: expected "
                         f"[N, {k // 2}] bytes")
    if scales.dtype != kind and scales.dtype != torch.uint8:
        raise ValueError(f"{fmt} scales are one byte each, {kind} or uint8; got {scales.dtype}")
    cols = k // block
    swizzle = scales.dim() == 1
    if swizzle and scales.numel() != -(-n // 128) * 128 * (-(-cols // 4)) * 4:
        raise ValueError(f"swizzled scales have {scales.numel()} bytes, expected "
                         f"{-(-n // 128) * 128 * (-(-cols // 4)) * 4}")
    if not swizzle and scales.shape != (n, cols):
        raise ValueError(f"expected scales [{n}, {cols}], got {tuple(scales.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), k)
    if x2.dtype not in nat.DTYPES:
        x2 = x2.float()
    m = x2.shape[0]
    if x2.stride(1) != 1 or (m > 1 and (x2.stride(0) % 8 or x2.stride(0) < k)) or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)  # also where x is contiguous and starts off 16 bytes
    c, s = codes.contiguous(), scales.contiguous()
    if c.data_ptr() % 8:
        c = c.clone()
    if s.data_ptr() % 4:
        s = s.clone()
    ts = tensor_scale
    if not isinstance(ts, torch.Tensor) or ts.dtype != torch.float32 or ts.get_device() != device \
            or not ts.is_contiguous():
        ts = torch.as_tensor(ts, dtype=torch.float32, device=x.device).contiguous()
    per_row = ts.numel() > 1
    if ts.numel() != (n if per_row else 1):
        raise ValueError(f"tensor_scale has {ts.numel()} values, expected 1 or {n}")
    if bias is None or (bias.dtype in nat.DTYPES and bias.shape == (n,) and bias.is_contiguous()):
        b, bias_code = bias, nat.KAB_F32 if bias is None else nat.DTYPES[bias.dtype]
    else:
        b, bias_code = _bias(bias, n, x.device)
    out = x2.new_empty((m, n))
    if k == 0:
        out.zero_()
        if b is not None:
            out += b
    elif m and n:
        dtype = nat.DTYPES[x2.dtype]
        stream = stream_of(device)
        nbytes = _plan(m, n, k, code, dtype, device)
        ws = workspace(device, nbytes) if nbytes else None
        call("kab_gemv_fp4", device, x2.data_ptr(), dtype, x2.stride(0) if m > 1 else k, c.data_ptr(), s.data_ptr(),
             swizzle, code, ts.data_ptr(), per_row, m, n, k, None if b is None else b.data_ptr(), bias_code,
             out.data_ptr(), n, None if ws is None else ws.data_ptr(), nbytes, stream)
    return out if out.dtype == x.dtype and x.dim() == 2 else q._linear_out(out, x, n)
