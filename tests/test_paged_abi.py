"""The paged cache's and the FP4 linear's C entry points without a GPU: struct layouts as the header
has them, and argument checks that fail before any launch."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from kernel_agent_b200 import _native as nat

ROOT = Path(__file__).resolve().parents[1]

pytestmark = pytest.mark.skipif(not nat.LIB_PATH.exists(), reason="libkab.so is not built")


@pytest.mark.parametrize("name", ["KabKvPages", "KabKvPagesAttention"])
def test_struct_layout(name, tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [f[0] for f in getattr(nat, name)._fields_]
    lines = "".join(f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "kab.h"\n'
                   f'int main(void) {{ printf("%zu\\n", sizeof({name})); {lines} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run([cc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    size, *offsets = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    mirror = getattr(nat, name)
    assert size == ctypes.sizeof(mirror)
    assert offsets == [getattr(mirror, f).offset for f in fields]


def pages(**kw) -> "nat.KabKvPages":
    p = nat.KabKvPages()
    p.k_pages = p.v_pages = p.k_scale = p.v_scale = p.mass = p.page_table = p.lengths = 256
    p.num_pages, p.heads_kv, p.page_tokens, p.head_dim, p.max_pages, p.batch, p.table_stride = 8, 2, 64, 128, 4, 1, 4
    p.k_stride_page = p.v_stride_page = 2 * 64 * 128
    p.k_stride_head = p.v_stride_head = 64 * 128
    p.k_stride_token = p.v_stride_token = 128
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,match", [
    ({"head_dim": 96}, "head_dim"), ({"page_tokens": 24}, "page_tokens"), ({"k_pages": 8}, "aligned"),
    ({"v_stride_token": 24}, "multiples of 16"), ({"k_stride_page": 1 << 31}, "2\\^31"), ({"lengths": None}, "lengths"),
    ({"page_table": None}, "page table"), ({"batch": -1}, "shape"), ({"heads_kv": 0}, "shape"),
    ({"max_pages": 1 << 25}, "too large"),
])
def test_append_checks(kw, match):
    p = pages(**kw)
    with pytest.raises(ValueError, match=match):
        nat.call("kab_kv_pages_append", ctypes.byref(p), 256, 256, nat.KAB_BF16, 256, 128, 128, 256, 128, 128, 1, None, 512, None)


def test_more_append_checks():
    p = pages()
    for args, match in (((256, 256, 9, 256, 128, 128, 256, 128, 128, 1, None, 512), "dtype"),
                        ((256, 256, 1, 256, 128, 12, 256, 128, 128, 1, None, 512), "multiples of 8"),
                        ((24, 256, 1, 256, 128, 128, 256, 128, 128, 1, None, 512), "aligned"),
                        ((256, 256, 1, 256, 128, 128, 256, 128, 128, -1, None, 512), "new tokens"),
                        ((256, 256, 1, 256, 128, 128, 256, 128, 128, 1, None, None), "lengths_out"),
                        ((None, 256, 1, 256, 128, 128, 256, 128, 128, 1, None, 512), "null")):
        with pytest.raises(ValueError, match=match):
            nat.call("kab_kv_pages_append", ctypes.byref(p), *args, None)


@pytest.mark.parametrize("budget,recent,sinks,mass,match", [
    (0, 0, 0, 256, "budget"), (8, 6, 3, 256, "budget"), (8, -1, 0, 256, "budget"), (8, 2, 2, None, "mass"),
])
def test_evict_checks(budget, recent, sinks, mass, match):
    p = pages(mass=mass)
    with pytest.raises(ValueError, match=match):
        nat.call("kab_kv_pages_evict", ctypes.byref(p), 256, 4, budget, recent, sinks, 256, 256, None)


def test_attention_checks():
    size = ctypes.c_size_t(0)
    for kw, match in (({"q_dtype": 7}, "dtype"), ({"heads_q": 3}, "multiple of heads_kv"), ({"q_len": -1}, "negative"),
                      ({"heads_q": 1 << 20, "q_len": 2}, "too many")):
        p = nat.KabKvPagesAttention()
        p.cache, p.q_dtype, p.heads_q, p.q_len = pages(), nat.KAB_BF16, 4, 1
        for k, v in kw.items():
            setattr(p, k, v)
        with pytest.raises(ValueError, match=match):
            nat.call("kab_kv_pages_attention_workspace", ctypes.byref(p), ctypes.byref(size))


def test_linear_checks():
    size = ctypes.c_size_t(0)
    for args, match in (((1, 8, 24, nat.KAB_NVFP4, 1), "multiple"), ((1, 8, 48, nat.KAB_MXFP4, 1), "multiple"),
                        ((1, 8, 32, 5, 1), "format"), ((1, 8, 32, 0, 8), "dtype"), ((-1, 8, 32, 0, 1), "negative"),
                        ((70000, 8, 32, 0, 1), "too large")):
        with pytest.raises(ValueError, match=match):
            nat.call("kab_gemv_fp4_workspace", *args, ctypes.byref(size))

    def run(x=256, ldx=32, codes=256, scales=256, ts=256, out=256, ldo=8):
        nat.call("kab_gemv_fp4", x, nat.KAB_BF16, ldx, codes, scales, 0, nat.KAB_NVFP4, ts, 0, 1, 8, 32, None, 0, out, ldo,
                 None, 0, None)

    for kw, match in (({"x": 8}, "aligned"), ({"ldx": 36}, "multiple of 8"), ({"codes": 4}, "8-byte"),
                      ({"scales": 258}, "4-byte"), ({"out": None}, "null"), ({"ts": None}, "null"), ({"ldo": 7}, "too short"),
                      ({"ldx": 24}, "too short")):
        with pytest.raises(ValueError, match=match):
            run(**kw)


def test_python_refuses_cpu_tensors():
    from kernel_agent_b200.kernels import gemv, paged_kv

    with pytest.raises(ValueError, match="CUDA tensor"):
        gemv.fp4_w4a16_linear(torch.zeros(1, 32), torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 1.0)
    pool = torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn)
    scale, table, lengths = torch.ones(2, 1), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged_kv.paged_kv_attention(torch.zeros(1, 1, 64), pool, scale, pool, scale, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        paged_kv.PagedFp8KVCache(1, 1, 64, 4, device="cpu")


def test_oracle_page_scale():
    """The smallest power of two that holds 448 times itself, to the ends of fp32."""
    from oracle import paged_kv as opk

    for amax, want in ((448.0, 1.0), (448.0001, 2.0), (0.0, 2.0 ** -126), (1e-45, 2.0 ** -126), (3.4e38, 2.0 ** 120),
                       (1.0, 2.0 ** -8), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7)):
        assert opk.page_scale(amax) == want
    kept = opk.keep(np.array([0.0, 5.0, 5.0, 1.0, 5.0, 9.0], np.float32), 6, 4, 1, 1)
    assert kept.tolist() == [0, 1, 2, 5]
