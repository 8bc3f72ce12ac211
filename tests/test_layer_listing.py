"""Compile-time check of the linear attention's listing for gfx950 (needs
hipcc, no GPU): no instruction meets an MFMA's result before it is there, on
any path (the scan of tests/test_mfma_waits.py)."""

from __future__ import annotations

import re
import shutil
from pathlib import Path

import pytest

from jeeves_amd import build
from tests.test_kernel_resources import compile_device
from tests.test_mfma_waits import early_uses, functions


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(), reason="needs hipcc")
def test_linear_attention_waits_for_its_products(tmp_path):
    _, asm = compile_device(build.CSRC / "linear_attention.hip", tmp_path)
    assert len(re.findall(r"^\s*v_mfma", asm, re.M)) > 500
    assert len(functions(asm)) > 10
    assert not early_uses(asm)
