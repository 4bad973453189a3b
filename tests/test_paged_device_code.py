"""Checks on the gfx950 device code of the paged attention kernels (CPU only): those of ``test_device_code.py`` for the
attention kernels, whose key-tile DMA these kernels share, and the packed FP32 forms that the build keeps out."""

import os
import re
import subprocess

import pytest

from sol_attn_amd import _build
from test_device_code import HIPCC, _sgpr_distances


@pytest.fixture(scope="module", params=["paged.hip", "cache.hip"])
def asm(request, tmp_path_factory):
    if HIPCC is None:
        pytest.skip("hipcc not installed")
    out = tmp_path_factory.mktemp("asm") / "out.s"
    cmd = [HIPCC, *_build.compile_flags(), "-Wno-inline-asm", "--cuda-device-only", "-S",
           os.path.join(_build.CSRC, request.param), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    assert res.returncode == 0, res.stderr[-2000:]
    return request.param, out.read_text().splitlines()


def test_only_the_key_tile_dma_uses_m0(asm):
    source, text = asm
    lines = [line.split(";")[0].strip() for line in text]
    code = [line for line in lines if line and not line.startswith(".") and not line.endswith(":")]
    writes = 0
    for i, line in enumerate(code):
        if re.search(r"\bm0\b", line):
            assert re.fullmatch(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)", line), f"unexpected use of M0: {line!r}"
            assert code[i + 1] == "s_nop 0" and code[i + 2].startswith("global_load_lds_dword")
            writes += 1
    assert (writes > 0) == (source == "paged.hip")


def test_inline_assembly_keeps_its_distance_from_vector_writes(asm):
    close = [(text, age) for text, inline, age in _sgpr_distances(asm[1])
             if inline and ((text.startswith("global_load_lds") and age < 5) or (text.startswith("v_") and age < 2))]
    assert not close, f"{len(close)}: {close[:4]!r}"


def test_no_packed_fp32(asm):
    assert not [line for line in asm[1] if re.search(r"\bv_pk_(add|mul|fma)_f32\b", line)]
