"""The weight-only FP4 linear on the GPU against the same sums in 64 bits.

Bound per element, with A = sum |x| |w| * tensor_scale: half a unit of the output type (2^-8,
2^-11 or 2^-24 of |y|, and fp16's smallest step), and an fp32 sum whose partial sums each lose at
most 2^-22 of A: at most K / 16 + 64 of them follow one another."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import np_bytes, np_values
from oracle import quant as oq

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
KINDS = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def gv():
    from kernel_agent_b200.kernels import gemv

    return gemv


def weight(n, k, fmt, seed=0):
    """Random codes with scales of a realistic spread: (codes, scales, values in 64 bits)."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    if fmt == "nvfp4":
        scales = torch.exp(torch.randn(n, k // 16, generator=g) * 1.5).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
        raw = np_bytes(scales)
    else:
        scales = torch.randint(110, 135, (n, k // 32), generator=g, dtype=torch.int32).to(torch.uint8)
        raw = scales.numpy()
        scales = scales.view(torch.float8_e8m0fnu)
    return codes.to(DEV), scales.to(DEV), oq.fp4_values(codes.numpy(), raw, fmt).astype(np.float64)


def check(y, x, w, ts, bias, dtype):
    xv = np_values(x).astype(np.float64)
    ts = np.asarray(ts, np.float64).reshape(1, -1)
    b = 0.0 if bias is None else np_values(bias).astype(np.float64)[None]
    want = (xv @ w.T) * ts + b
    size = (np.abs(xv) @ np.abs(w).T) * np.abs(ts) + np.abs(b)
    tol = UNIT[dtype] * np.abs(want) + (w.shape[1] / 16 + 64) * 2.0 ** -22 * size + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    assert np.all(np.abs(np_values(y) - want) <= tol)


SHAPES = [(1, 1, 32), (1, 16, 64), (2, 17, 96), (3, 200, 4128), (1, 1024, 1024), (8, 129, 512), (9, 64, 2080),
          (16, 300, 256), (17, 40, 8192), (32, 1001, 4096), (33, 16, 1024), (7, 24, 14336), (1, 5000, 288), (100, 48, 320)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear(gv, shape, dtype, fmt):
    m, n, k = shape
    codes, scales, w = weight(n, k, fmt, m)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(m, k, generator=g).to(dtype).to(DEV)
    ts = 0.003 if fmt == "nvfp4" else 1.0 / 256  # keeps fp16 outputs in range
    bias = torch.randn(n, generator=g).to(dtype).to(DEV) if n % 2 else None
    y = gv.fp4_w4a16_linear(x, codes, scales, torch.tensor(ts, device=DEV), bias, fmt=fmt)
    assert y.dtype == dtype and y.shape == (m, n)
    check(y, x, w, np.float32(ts), bias, dtype)
    assert torch.equal(y, gv.fp4_w4a16_linear(x, codes, scales, torch.tensor(ts, device=DEV), bias, fmt=fmt))
    flat = torch.from_numpy(oq.swizzle_scales(np_bytes(scales))).to(DEV)
    y = gv.fp4_w4a16_linear(x, codes, flat, torch.tensor(ts, device=DEV), bias, fmt=fmt)
    check(y, x, w, np.float32(ts), bias, dtype)


@pytest.mark.parametrize("dtype", KINDS)
def test_nvfp4_odd_blocks(gv, dtype):
    """K a multiple of 16 and not of 32, one block alone among them; codes off a 16-byte boundary."""
    for m, n, k in ((1, 5, 16), (4, 33, 48), (8, 130, 4080), (2, 64, 8176)):
        codes, scales, w = weight(n, k, "nvfp4", k)
        x = torch.randn(m, k, device=DEV).to(dtype)
        check(gv.fp4_w4a16_linear(x, codes, scales, 0.01), x, w, np.float32(0.01), None, dtype)
    codes, scales, w = weight(17, 48, "nvfp4", 1)
    check(gv.fp4_w4a16_linear(x[:, :48], codes[1:], scales[1:], 0.01), x[:, :48], w[1:], np.float32(0.01), None, dtype)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wide_ranges(gv, fmt, dtype):
    """Activations and scales over the whole range of their types: each product counts by its own
    size, whatever stands beside it."""
    n, k = 48, 1024
    codes, scales, _ = weight(n, k, fmt, 9)
    g = torch.Generator().manual_seed(4)
    if fmt == "nvfp4":
        raw = torch.randint(0, 0x7F, (n, k // 16), generator=g, dtype=torch.int32).to(torch.uint8)
        scales = raw.view(torch.float8_e4m3fn).to(DEV)
    else:
        raw = torch.randint(60, 190, (n, k // 32), generator=g, dtype=torch.int32).to(torch.uint8)
        scales = raw.view(torch.float8_e8m0fnu).to(DEV)
    w = oq.fp4_values(codes.cpu().numpy(), raw.numpy(), fmt).astype(np.float64)
    x = (torch.randn(4, k, generator=g) * torch.logspace(-3, 1, 4)[:, None] * torch.logspace(0, 6, k)).to(dtype).to(DEV)
    check(gv.fp4_w4a16_linear(x, codes, scales, 0.5, fmt=fmt), x, w, 0.5, None, dtype)
    x = (x.float() * 1e25).to(dtype)
    check(gv.fp4_w4a16_linear(x, codes, scales, 1e-30, fmt=fmt), x, w, np.float32(1e-30), None, dtype)
    x = (x.float() * 1e-50).to(dtype)
    check(gv.fp4_w4a16_linear(x, codes, scales, 1e20, fmt=fmt), x, w, np.float32(1e20), None, dtype)


def test_mxfp4_far_scales(gv):
    """A block of zeros may carry any scale; blocks 2^100 apart keep their own products."""
    codes, scales, _ = weight(16, 128, "mxfp4", 2)
    raw = torch.full((16, 4), 27, dtype=torch.uint8)
    raw[:, 2] = 200
    codes = codes.clone()
    codes[:, 32:48] = 0
    w = oq.fp4_values(codes.cpu().numpy(), raw.numpy(), "mxfp4").astype(np.float64)
    x = torch.randn(1, 128, device=DEV)
    y = gv.fp4_w4a16_linear(x, codes, raw.view(torch.float8_e8m0fnu).to(DEV), 2.0 ** 99, fmt="mxfp4")
    check(y, x, w, 2.0 ** 99, None, torch.float32)


@pytest.mark.parametrize("dtype", KINDS)
def test_nonfinite(gv, dtype):
    """An infinity or NaN in one row of x reaches that row's outputs alone; a NaN scale its row of W."""
    codes, scales, w = weight(32, 256, "nvfp4", 3)
    codes = (codes & 0x77) | 0x11  # every value positive
    x = torch.rand(4, 256, device=DEV).to(dtype) + 0.5
    x[1, 7], x[2, 200] = float("inf"), float("nan")
    y = gv.fp4_w4a16_linear(x, codes, scales, 0.01).float()
    assert torch.isposinf(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()
    bad = scales.clone()
    bad.view(torch.uint8)[5, 3] = 0x7F
    y = gv.fp4_w4a16_linear(x[:1], codes, bad, 0.01).float()
    assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()


def test_tensor_scales_bias_and_strides(gv):
    codes, scales, w = weight(80, 512, "nvfp4", 6)
    x = torch.randn(2, 3, 1, 520, device=DEV).to(torch.bfloat16)[..., 4:516]  # off 16 bytes
    ts = torch.rand(80, device=DEV) * 0.01
    bias = torch.randn(80, device=DEV, dtype=torch.float64)
    y = gv.fp4_w4a16_linear(x, codes, scales, ts, bias)
    assert y.shape == (2, 3, 1, 80)
    check(y.reshape(6, 80), x.reshape(6, 512), w, ts.cpu().numpy(), bias, torch.bfloat16)
    wide = torch.randn(4, 2, 512, device=DEV).to(torch.float16)
    check(gv.fp4_w4a16_linear(wide[:, 1], codes, scales, 0.001), wide[:, 1], w, np.float32(0.001), None, torch.float16)
    assert gv.fp4_w4a16_linear(x[:0], codes, scales, ts).shape == (0, 3, 1, 80)
    same = wide[:1, 1].expand(5, 512)  # one row five times
    check(gv.fp4_w4a16_linear(same, codes, scales, 0.001), same, w, np.float32(0.001), None, torch.float16)
    none = gv.fp4_w4a16_linear(x[..., :0], codes[:, :0], scales[:, :0], ts, bias)
    assert torch.equal(none, bias.to(torch.bfloat16).expand(2, 3, 1, 80))


def test_same_weight_as_w4a4(gv):
    """One quantised weight serves both linears."""
    from kernel_agent_b200.kernels import quant

    w = torch.randn(256, 512, device=DEV) * 0.02
    x = torch.randn(5, 512, device=DEV).to(torch.bfloat16)
    for fmt in ("nvfp4", "mxfp4"):
        codes, scales, ts = quant.quantize_fp4(w.to(torch.bfloat16), fmt)
        y = gv.fp4_w4a16_linear(x, codes, scales, ts, fmt=fmt)
        check(y, x, np_values(quant.fp4_values(codes, scales)).astype(np.float64), ts.cpu().numpy(), None, torch.bfloat16)
        both = quant.fp4_w4a4_linear(x, codes, scales, ts, fmt=fmt)
        assert float((y.float() - both.float()).norm() / y.float().norm()) < 0.2  # W4A4 also rounds x


def test_streams_and_graphs(gv):
    codes, scales, _ = weight(512, 8192, "nvfp4", 8)
    x = torch.randn(2, 8192, device=DEV).to(torch.bfloat16)
    ts = torch.tensor(0.01, device=DEV)
    want = gv.fp4_w4a16_linear(x, codes, scales, ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gv.fp4_w4a16_linear(x, codes, scales, ts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gv.fp4_w4a16_linear(x, codes, scales, ts)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_refusals(gv):
    codes, scales, _ = weight(32, 256, "nvfp4", 3)
    x = torch.randn(1, 256, device=DEV)
    for args, kw, match in (
        ((x.cpu(), codes, scales, 1.0), {}, "CUDA tensor"),
        ((x, codes, scales, 1.0), {"fmt": "int4"}, "unknown FP4 format"),
        ((x[:, :250], codes, scales, 1.0), {}, "multiple"),
        ((x[:, :128], codes, scales, 1.0), {}, "fit"),
        ((x, codes, scales[:, :8], 1.0), {}, "scales"),
        ((x, codes, scales.float(), 1.0), {}, "one byte"),
        ((x, codes, scales.view(torch.float8_e8m0fnu), 1.0), {}, "nvfp4 scales"),
        ((x, codes, scales[:, ::2].contiguous(), 1.0), {"fmt": "mxfp4"}, "mxfp4 scales"),
        ((x, codes, scales.reshape(-1), 1.0), {}, "swizzled"),
        ((x, codes, scales, torch.ones(3, device=DEV)), {}, "tensor_scale"),
        ((x, codes, scales, 1.0, torch.ones(31, device=DEV)), {}, "bias"),
    ):
        with pytest.raises(ValueError, match=match):
            gv.fp4_w4a16_linear(*args, **kw)
