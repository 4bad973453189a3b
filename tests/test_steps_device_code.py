"""Checks on the gfx950 device code of the rotation and of the cache's steps (CPU only): none of the packed FP32 forms
that the build keeps out, and no memory of their own per lane (the compiler may hold a lane's arrays in LDS)."""

import os
import re
import subprocess

import pytest

from sol_attn_amd import _build
from test_device_code import HIPCC


@pytest.mark.parametrize("source", ["rotate.hip", "fork.hip"])
def test_no_packed_fp32_and_no_scratch(source, tmp_path):
    if HIPCC is None:
        pytest.skip("hipcc not installed")
    out = tmp_path / "out.s"
    cmd = [HIPCC, *_build.compile_flags(), "--cuda-device-only", "-S", os.path.join(_build.CSRC, source), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    assert not re.search(r"^\s+scratch_(load|store)", text, re.M)
    if source == "rotate.hip":
        assert set(re.findall(r"amdhsa_group_segment_fixed_size (\d+)", text)) == {"0"}
