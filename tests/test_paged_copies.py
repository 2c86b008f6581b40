"""Wait states of the paged decode's HBM -> LDS copies in the compiled kernels, as in test_lds_dma_hazards (CPU only, needs hipcc)."""
import os
import subprocess

import pytest

from test_lds_dma_hazards import HIPCC, PKG, dma_hazards


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_paged_decode_wait_states(tmp_path):
    # the Makefile's own line for this source, to assembly
    line = subprocess.run(["make", "-n", "-B", "_build/decode_paged.o"], cwd=PKG, capture_output=True, text=True, check=True).stdout
    line = [l for l in line.splitlines() if "decode_paged.hip" in l][0].split()
    out = tmp_path / "decode_paged.s"
    cmd = [HIPCC] + line[1:line.index("-c")] + ["--offload-device-only", "-S", "csrc/decode_paged.hip", "-o", str(out)]
    r = subprocess.run(cmd, cwd=PKG, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = out.read_text().split("\n")
    assert any(l.strip().startswith("global_load_lds") for l in lines)
    bad = dma_hazards(lines)
    assert not bad, f"{len(bad)} LDS DMA(s) without 5 wait states after a VALU SGPR write, e.g. {bad[:3]}"
    assert not any("v_pk_fma_f32" in l or "v_pk_mul_f32" in l or "v_pk_add_f32" in l for l in lines)
