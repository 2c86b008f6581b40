"""The packed prompts' plan (csrc/packed_plan.hpp), swept on the CPU: size 0 means the same kernel with and without a
workspace, and other sizes hold what the kernels store."""
import os
import subprocess

import pytest

import cdna4

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")


def test_plans_with_and_without_a_workspace():
    subprocess.run(["make", "-C", NATIVE, "packed_plan_check"], check=True, capture_output=True)
    r = subprocess.run([os.path.join(NATIVE, "packed_plan_check")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    seen, ok = r.stdout.split("\n")[:2]
    assert ok == "ok" and all(int(n) > 0 for n in seen.split())      # dealt out, listed, cut


@pytest.mark.parametrize("D,total,prefix", [(128, 1008, 4096), (128, 1008, 8960), (64, 791, 8192)])
def test_reported_blocks_are_those_of_the_call(D, total, prefix):
    """One prompt whose blocks are not cut: the half blocks that a call without a workspace runs (on 256 CUs)."""
    cfg = cdna4.PackedPrefillCfg(D, 32, 8, 1, total, total, prefix, 0)
    p = cdna4.prefill_packed_plan(cfg)
    assert p.workspace == 0 and p.rows == 16
