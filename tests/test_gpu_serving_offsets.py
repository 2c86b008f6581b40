"""The batched serving calls where element offsets pass 32 bits: rows, heads and sequences far apart in memory. What
lies between them is never written and holds whatever the allocator left."""
import pytest
import torch

import cdna4
from serving_util import DEV, check, cu_of, packed_reference, shared_reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return lambda dtype, *s: torch.randn(*s, device=DEV, generator=g).to(dtype)


@pytest.mark.parametrize("row,lens,prefix", [
    (1 << 20, [1500, 0, 640], 0),      # the last rows begin past 2^31 elements; a tile's rows within 4 GiB
    (1 << 24, [100, 1, 40], 0),        # a tile's rows past 4 GiB
    (1 << 24, [100, 1, 40], 1100),     # behind a prefix, cut along the keys
])
def test_packed_rows_far_apart(row, lens, prefix):
    rnd = gen(prefix + row)
    HQ, HK, D, T = 8, 2, 128, sum(lens)
    x = torch.empty((T - 1) * row + (HQ + 2 * HK) * D, dtype=BF16, device=DEV)
    Q, K, V = (x[o * D:].as_strided((T, h, D), (row, D, 1)) for o, h in ((0, HQ), (HQ, HK), (HQ + HK, HK)))
    for t in (Q, K, V):
        t.copy_(rnd(BF16, *t.shape))
    Kp = Vp = None
    if prefix:
        Kp, Vp = rnd(BF16, HK, prefix, D), rnd(BF16, HK, prefix, D)
    cu = cu_of(lens)
    cfg = cdna4.PackedPrefillCfg(D, HQ, HK, len(lens), T, 0, prefix, 0)
    assert (cdna4.prefill_packed_workspace_size(cfg) > 0) == (prefix > 0)
    y = torch.empty((T - 1) * row + HQ * D, dtype=BF16, device=DEV)
    O = y.as_strided((T, HQ, D), (row, D, 1))
    cdna4.prefill_packed(Q, K, V, O, torch.tensor(cu, dtype=torch.int32, device=DEV), cfg, Kp, Vp)
    ref, bound, _ = packed_reference(Q.contiguous(), K.contiguous(), V.contiguous(), cu, D, HQ // HK, BF16, Kp, Vp, prefix)
    check(O, ref, bound)


def test_shared_heads_and_sequences_far_apart():
    """The prefix's last kv head and the last sequences' caches begin past 2^31 elements."""
    rnd = gen(5)
    HQ, HK, D, P, far = 16, 4, 128, 300, 6_000_000
    B, rows = 33, 145_000
    lens = [0] * (B - 3) + [77, 200, 1]
    x = torch.empty(2, HK, far, D, dtype=F16, device=DEV)
    own = torch.empty(2, B, HK, rows, D, dtype=F16, device=DEV)
    assert (HK - 1) * far * D > 2 ** 31 and (B - 3) * HK * rows * D > 2 ** 31
    x[:, :, :P] = rnd(F16, 2, HK, P, D)
    for b in range(B - 3, B):
        own[:, b, :, :lens[b]] = rnd(F16, 2, HK, lens[b], D)
    q = rnd(F16, B, HQ, D)
    cfg = cdna4.SharedDecodeCfg(D, HQ, HK, B, P, far, 256, rows)
    o = torch.empty_like(q)
    cdna4.decode_shared(q, x[0], x[1], own[0], own[1], torch.tensor(lens, dtype=torch.int32, device=DEV), o, cfg)
    ref, bound = shared_reference(q, x[0], x[1], own[0], own[1], lens, HQ // HK, F16, P)
    check(o, ref, bound)


def test_logits_rows_far_apart():
    """Equal bits to the same rows side by side."""
    rnd = gen(6)
    M, V, far = 3, 1003, (1 << 30) + 1
    kw = dict(history=torch.randint(0, V, (M, 50), device=DEV, dtype=torch.int32), repetition=torch.full((M,), 1.3, device=DEV),
              frequency=torch.full((M,), 0.2, device=DEV))
    near = rnd(F16, M, V)
    x = torch.empty((M - 1) * far + V, dtype=F16, device=DEV).as_strided((M, V), (far, 1))
    y = torch.empty((M - 1) * far + V, dtype=torch.float32, device=DEV).as_strided((M, V), (far, 1))
    x.copy_(near)
    cdna4.process_logits(x, y, **kw)
    assert torch.equal(y, cdna4.process_logits(near, **kw))
