"""Test files give the same results in any order."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

from kernel_agent_b200 import _native as nat

TESTS = Path(__file__).resolve().parent


@pytest.mark.skipif(not nat.LIB_PATH.exists(), reason="libkab.so is not built")
def test_refusals_before_the_library_metadata():
    """Refusals leave their message as the library's last error; the check that a fresh library has none runs
    before them."""
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", "-k",
                        "more_append_checks or metadata", str(TESTS / "test_paged_abi.py"), str(TESTS / "test_abi.py")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "2 passed" in r.stdout, r.stdout[-2000:]
