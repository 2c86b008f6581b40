"""cdna4.decode_shared against a 64-bit reference: prefixes and own caches from no key to several parts, odd
lengths, head layouts, batches of more rows than a block, lengths read on the device."""
import pytest
import torch

import cdna4
from serving_util import DEV, check, shared_reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(lens, HQ, HK, D, dtype, prefix, cap=None, room=(3, 2), seed=0, scale=1.0):
    """Own rows from each length on and prefix rows behind the prefix hold NaN: they must not reach a result."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)
    B = len(lens)
    cap = max(lens) if cap is None else cap
    q = (rnd(B, HQ, D) * scale).to(dtype)
    Kp = Vp = K = V = lens_d = None
    if prefix:
        Kp, Vp = rnd(HK, prefix + room[0], D), rnd(HK, prefix + room[0], D)
        Kp[:, prefix:], Vp[:, prefix:] = float("nan"), float("nan")
    if cap:
        K, V = rnd(B, HK, cap + room[1], D), rnd(B, HK, cap + room[1], D)
        for b, n in enumerate(lens):
            K[b, :, n:], V[b, :, n:] = float("nan"), float("nan")
        lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cfg = cdna4.SharedDecodeCfg(D, HQ, HK, B, prefix, prefix + room[0] if prefix else 0, cap, cap + room[1] if cap else 0)
    return q, Kp, Vp, K, V, lens_d, cfg


def run(q, Kp, Vp, K, V, lens_d, cfg, o=None, **kw):
    o = torch.full_like(q, 7.0) if o is None else o
    cdna4.decode_shared(q, Kp, Vp, K, V, lens_d, o, cfg, **kw)
    return o


def verify(args, lens, o, what=""):
    q, Kp, Vp, K, V, _, cfg = args
    ref, bound = shared_reference(q, Kp, Vp, K, V, lens, cfg.nQHeads // cfg.nKVHeads, q.dtype, cfg.prefix)
    return check(o, ref, bound, what)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [0, 1, 31, 33, 63, 64, 65, 127, 128, 129, 200, 1000, 1531])
def test_prefixes(prefix, D, dtype):
    lens = [0, 1, 31, 32, 33, 64, 65, 100, 300]
    args = make(lens, 8, 2, D, dtype, prefix, seed=prefix)
    verify(args, lens, run(*args), f"prefix {prefix}")


@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 0], [700], [1, 0, 2047, 5], [64] * 7])
@pytest.mark.parametrize("prefix", [0, 77])
@pytest.mark.parametrize("D", [64, 128])
def test_own_lengths(lens, prefix, D):
    args = make(lens, 4, 4, D, BF16, prefix, cap=max(max(lens), 1), seed=len(lens))
    o = run(*args)
    verify(args, lens, o)
    if prefix == 0:
        for b, n in enumerate(lens):
            if n == 0:
                assert bool((o[b] == 0).all())     # a row that sees nothing


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (16, 2), (40, 8), (12, 12), (20, 1), (33, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(heads, D):
    lens = [70, 0, 129]
    args = make(lens, *heads, D, F16, 150, seed=heads[0])
    verify(args, lens, run(*args))


@pytest.mark.parametrize("B", [1, 2, 31, 32, 33, 64, 65, 130])
def test_batches(B):
    """Rows per kv head (4 B) below, at and past a block of 128."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    args = make(lens, 4, 1, 128, BF16, 333, cap=90, seed=B)
    verify(args, lens, run(*args))


def test_prefix_alone():
    args = make([0] * 5, 8, 2, 128, F16, 500, cap=0, seed=1)
    assert args[3] is None
    verify(args, None, run(*args))


def test_no_keys_at_all():
    args = make([0] * 3, 8, 2, 64, F16, 0, cap=0)
    assert bool((run(*args) == 0).all())


def test_long():
    """Several parts of several tiles on both sides, the loops' steady state."""
    lens = [4000, 17, 9000, 0, 2500]
    for D, dtype in ((128, BF16), (64, F16)):
        args = make(lens, 16, 4, D, dtype, 20011, cap=9001, seed=2)
        verify(args, lens, run(*args))


def test_more_keys_than_parts():
    """A capacity far above the lengths, and lengths at the capacity."""
    lens = [3, 40000, 100]
    args = make(lens, 2, 1, 64, F16, 10, cap=40000, seed=3)
    verify(args, lens, run(*args))


@pytest.mark.parametrize("scale", [0.0, 8.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_peaked_and_flat(scale, dtype):
    lens = [300, 0, 64]
    args = make(lens, 8, 2, 128, dtype, 700, seed=4, scale=scale)
    verify(args, lens, run(*args))


def test_lengths_are_cut():
    lens = [-5, 1000, 2 ** 31 - 1, -2 ** 31, 60]
    args = make([0, 100, 100, 0, 60], 4, 2, 64, F16, 50, cap=100, seed=5)
    args[5].copy_(torch.tensor(lens, dtype=torch.int32))
    verify(args, [0, 100, 100, 0, 60], run(*args))


def test_as_decode_where_lengths_are_equal():
    lens = [777] * 3
    q, _, _, K, V, lens_d, cfg = make(lens, 8, 2, 128, BF16, 0, room=(0, 0), seed=6)
    o = run(q, None, None, K, V, lens_d, cfg)
    u = torch.empty_like(q)
    cdna4.decode(q, K, V, u, cdna4.DecodeCfg(128, 777, 8, 2, 3, 0))
    _, bound = shared_reference(q, None, None, K, V, lens, 4, BF16)
    check(o, u.double(), 2 * bound)


def test_workspace_contents_do_not_matter():
    lens = [40, 0, 200]
    args = make(lens, 8, 2, 128, F16, 300, seed=7)
    need = cdna4.decode_shared_workspace_size(args[-1])
    a = run(*args)
    for fill in (0, 255):
        ws = torch.full((need + 64,), fill, dtype=torch.uint8, device=DEV)
        assert torch.equal(a, run(*args, workspace=ws[:need]))
        assert bool((ws[need:] == fill).all())
    with pytest.raises(cdna4.CDNA4Error):
        run(*args, workspace=ws[:need - 1])
    for bad in (None, "none"):
        with pytest.raises(ValueError):
            run(*args, workspace=bad)


def test_two_streams_at_once():
    la, lb = [400, 30, 0], [77, 500]
    a = make(la, 8, 2, 128, BF16, 1000, seed=8)
    b = make(lb, 12, 12, 64, F16, 90, seed=9)
    oa, ob = torch.empty_like(a[0]), torch.empty_like(b[0])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        run(*a, o=oa, stream=s1)
        run(*b, o=ob, stream=s2)
    torch.cuda.synchronize()
    verify(a, la, oa)
    verify(b, lb, ob)


def test_captured_call_replays_on_other_lengths():
    cap = 600
    q, Kp, Vp, K, V, lens_d, cfg = make([cap] * 4, 8, 2, 128, F16, 130, cap=cap, seed=10)
    ws = torch.empty(cdna4.decode_shared_workspace_size(cfg), dtype=torch.uint8, device=DEV)
    o = torch.empty_like(q)
    run(q, Kp, Vp, K, V, lens_d, cfg, o=o, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(q, Kp, Vp, K, V, lens_d, cfg, o=o, workspace=ws)
    for lens in ([0, 0, 0, 0], [1, 600, 33, 64], [599, 2, 0, 300], [600] * 4):
        lens_d.copy_(torch.tensor(lens, dtype=torch.int32))
        o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, run(q, Kp, Vp, K, V, lens_d, cfg))
        verify((q, Kp, Vp, K, V, lens_d, cfg), lens, o, str(lens))
