"""What a cut call of cdna4.prefill_packed leaves in its workspace for the join: how many items were cut and how, and in
each cut item's place the item itself, whichever wave of a workgroup looked it up."""
import pytest
import torch

import cdna4
from serving_util import DEV
from test_gpu_prefill_packed import CUT, UNCUT, make, run, verify

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16

ROUNDS = {"more_than_a_round": 1, "a_round_and_more": 1, "round_of_half_blocks": 1, "a_round_and_few": 1}   # of 256 CUs
UNUSED = "reserved_only"   # sizes that may need a cut, lengths that do not
CASES = {n: c for n, c in CUT.items() if n not in UNCUT} | {UNUSED: ([40] * 20, 32, 8, 128, BF16, 2048)}


def items_of(lens, rows, heads_per, HQ):
    """(first row, rows, first query, first head) of every item, in the order they are dealt out in: last blocks first,
    sequences ascending within one index; the heads of an entry in any order."""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    most = max(-(-n // rows) for n in lens)
    return [{(cu[s], n, d * rows, h * heads_per) for h in range(HQ // heads_per)}
            for d in range(most - 1, -1, -1) for s, n in enumerate(lens) if -(-n // rows) > d]


@pytest.mark.parametrize("name", sorted(CASES))
def test_places_of_the_cut_items(name):
    lens, HQ, HK, D, dtype, prefix = CASES[name]
    args = make(lens, HQ, HK, D, dtype, prefix=prefix, spare=2, seed=len(lens))
    cfg = args[-1]
    plan = cdna4.prefill_packed_plan(cfg, dtype)
    per = 4 if (HQ // HK) % 4 == 0 else 2 if (HQ // HK) % 2 == 0 else 1
    entries = items_of(lens, plan.rows, per, HQ)
    nh, total = HQ // per, len(entries) * (HQ // per)
    ws = torch.full((plan.workspace,), 255, dtype=torch.uint8, device=DEV)
    O = run(*args[:5], *args[6:], workspace=ws)
    rounds, tail, each = ws[:12].view(torch.int32).tolist()
    assert rounds == total // plan.grid
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert rounds == ROUNDS.get(name, 0) and (tail > 0) == (name != UNUSED)
    if tail:
        assert tail == total % plan.grid and 2 <= each <= 32 and each * tail <= plan.grid
        got = [tuple(x) for x in ws[256:256 + 16 * tail].view(torch.int32).view(tail, 4).tolist()]
        assert len(set(got)) == tail
        for e, item in enumerate(got):
            assert item in entries[(rounds * plan.grid + e) // nh], (e, item)
    verify(args, cfg, dtype, O, name)
    for _ in range(3):
        assert torch.equal(O, run(*args[:5], *args[6:], workspace=ws))


@pytest.mark.parametrize("D,total,prefix", [(128, 1008, 4096), (128, 1008, 8960), (64, 791, 8192)])
def test_workspace_of_a_call_that_needs_none(D, total, prefix):
    """Where the size is 0, a caller's workspace changes no bit and is not written to."""
    args = make([total], 32, 8, D, BF16, prefix=prefix, seed=prefix)
    assert cdna4.prefill_packed_workspace_size(args[-1]) == 0
    ws = torch.full((4096,), 255, dtype=torch.uint8, device=DEV)
    one = run(*args[:5], *args[6:], workspace=None)
    assert torch.equal(one, run(*args[:5], *args[6:], workspace=ws)) and torch.equal(one, run(*args[:5], *args[6:]))
    assert bool((ws == 255).all())
    verify(args, args[-1], BF16, one)
