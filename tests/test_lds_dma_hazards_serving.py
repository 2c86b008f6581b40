"""The wait-state check of test_lds_dma_hazards for the batched serving kernels: every LDS DMA's scalar operands are
moved by the SALU, and no copy's base ended in a vector register (its asm could not take it)."""
import os
import re
import subprocess

import pytest

from test_lds_dma_hazards import HIPCC, PKG, dma_hazards

SOURCES = ["prefill_packed.hip", "decode_shared.hip"]


def flags():
    """HIPFLAGS as the Makefile has them, with the scheduler that it sets for these sources."""
    mk = open(os.path.join(PKG, "Makefile")).read()
    for src in SOURCES:
        assert re.search(r"_build/%s[^\n]*HIPFLAGS \+= -mllvm -amdgpu-sched-strategy=iterative-ilp" % src.replace(".hip", r"\.o"), mk), src
    return ["--offload-arch=gfx950", "-O3", "-std=c++17", "-I../include", "-Icsrc", "-Xclang", "-target-feature", "-Xclang",
            "-packed-fp32-ops", "-Wno-unused-command-line-argument", "-mllvm", "-amdgpu-sched-strategy=iterative-ilp"]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("src", SOURCES)
def test_lds_dma_wait_states(src, tmp_path):
    out = tmp_path / (src + ".s")
    r = subprocess.run([HIPCC] + flags() + ["--offload-device-only", "-S", os.path.join("csrc", src), "-o", str(out)], cwd=PKG,
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = out.read_text().split("\n")
    assert sum(1 for l in lines if l.strip().startswith("global_load_lds")) > 0
    bad = dma_hazards(lines)
    assert not bad, f"{len(bad)} LDS DMA(s) without 5 wait states after a VALU SGPR write, e.g. {bad[:3]}"
    assert not any(re.search(r"s_mov_b64 s\[\d+:\d+\], v\[", l) for l in lines)
    assert not any(re.search(r"v_pk_(add|mul|fma)_f32", l) for l in lines)
