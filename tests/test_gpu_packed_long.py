"""cdna4.prefill_packed on sequences of more than 1,024 blocks, past what a workgroup holds of the block counts: a row of
every block against the 64-bit reference, every row written, and the same bits however the blocks are handed out."""
import pytest
import torch

import cdna4
from serving_util import DEV, attend, check
from test_gpu_prefill_packed import make, run

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
LEVELS = 1024

CASES = {   # tokens, heads, D, type, prefix, whether a workspace lists the blocks
    "dealt": ([33500, 5, 0, 32900, 100, 32768, 32769], 4, 1, 64, F16, 0, False),
    "dealt_prefix": ([32801, 700, 33333], 4, 1, 64, BF16, 777, False),
    "pairs": ([65600, 64, 1], 2, 1, 64, F16, 0, False),
    "one_head": ([131300, 129], 1, 1, 64, F16, 0, False),
    "listed": ([100, 33500, 5, 32900, 0, 32768, 34000, 1], 8, 2, 128, BF16, 0, True),
    "listed_prefix": ([32801, 700, 33333], 4, 1, 128, F16, 1025, True),
    "batch": ([3] * 600 + [33000] + [40] * 100 + [32770], 4, 1, 64, F16, 0, False),     # past the rows held as well
}


@pytest.mark.parametrize("name", list(CASES))
def test_more_blocks_than_levels(name):
    lens, HQ, HK, D, dtype, prefix, listed = CASES[name]
    Q, K, V, Kp, Vp, cu, cu_d, cfg = make(lens, HQ, HK, D, dtype, prefix=prefix, spare=2, seed=len(lens))
    rows = cdna4.prefill_packed_plan(cfg, dtype).rows
    assert sum(-(-n // rows) > LEVELS for n in lens) >= (1 if name in ("pairs", "one_head") else 2)
    assert (cdna4.prefill_packed_workspace_size(cfg) > 0) == listed
    one = run(Q, K, V, Kp, Vp, cu_d, cfg, workspace=None)
    if listed:
        assert torch.equal(one, run(Q, K, V, Kp, Vp, cu_d, cfg))
    T = cu[-1]
    assert bool((one[T:] == 7.0).all()), "rows of no sequence were written"
    assert not bool((one[:T] == 7.0).all(-1).any()), "rows of a sequence were not written"
    g = torch.Generator().manual_seed(len(lens))
    for s, n in enumerate(lens):
        if n == 0 or (n < 1000 and s > 8):
            continue
        starts = torch.arange(0, n, rows)
        at = starts + (torch.rand(len(starts), generator=g) * (n - starts).clamp(max=rows)).long()
        at = torch.cat([at, torch.tensor([0, n - 1])]).to(DEV)
        a, G = cu[s], HQ // HK
        seen = torch.arange(prefix + n, device=DEV)[None] <= prefix + at[:, None]
        for h in range(HQ):
            k, v = K[a:a + n, h // G], V[a:a + n, h // G]
            if prefix:
                k, v = torch.cat([Kp[h // G, :prefix], k]), torch.cat([Vp[h // G, :prefix], v])
            for i in range(0, len(at), 256):
                ref, bound = attend(Q[a + at[i:i + 256], h], k, v, seen[i:i + 256], dtype)
                check(one[a + at[i:i + 256], h], ref, bound, f"sequence {s}, head {h}")
