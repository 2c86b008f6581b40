"""How packed prompts' items are dealt out and cut along their keys (csrc/packed_cut.hpp), replayed on the CPU: every
item and part once, and one store to each place that the join reads."""
import os
import subprocess

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")


def test_every_item_and_part_is_taken_once():
    subprocess.run(["make", "-C", NATIVE, "packed_cut_check"], check=True, capture_output=True)
    r = subprocess.run([os.path.join(NATIVE, "packed_cut_check")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    cuts, ok = r.stdout.split("\n")[:2]
    assert ok == "ok" and all(int(n) > 0 for n in cuts.split())      # cuts after 0, 1, 2, 3 and more whole rounds
