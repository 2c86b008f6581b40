"""Packed prompts (cdna4.prefill_packed) against a 64-bit reference: lengths from none to several blocks, odd
ones, prefixes that end anywhere in a tile, head layouts, strides, lengths read on the device."""
import pytest
import torch

import cdna4
from serving_util import DEV, check, cu_of, packed_reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(lens, HQ, HK, D, dtype, prefix=0, spare=0, first=0, seed=0, layout="fused", room=5, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)
    T = first + sum(lens) + spare
    if layout == "fused":       # Q, K and V side by side per token
        x = rnd(T, HQ + 2 * HK, D)
        Q, K, V = x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:]
    elif layout == "heads":     # head-major storage
        Q, K, V = (rnd(h, T, D).transpose(0, 1) for h in (HQ, HK, HK))
    elif layout == "wide":      # rows longer than D
        Q, K, V = (rnd(T, h, D + 8)[..., :D] for h in (HQ, HK, HK))
    else:
        Q, K, V = rnd(T, HQ, D), rnd(T, HK, D), rnd(T, HK, D)
    Q = Q * scale if scale != 1.0 else Q
    Kp = Vp = None
    if prefix:
        Kp, Vp = rnd(HK, prefix + room, D), rnd(HK, prefix + room, D)
        Kp[:, prefix:], Vp[:, prefix:] = float("nan"), float("nan")    # behind the prefix: never read into a result
    cu = cu_of(lens, first)
    cfg = cdna4.PackedPrefillCfg(D, HQ, HK, len(lens), T, max(lens, default=0), prefix, prefix + room if prefix else 0)
    return Q, K, V, Kp, Vp, cu, torch.tensor(cu, dtype=torch.int32, device=DEV), cfg


def run(Q, K, V, Kp, Vp, cu_d, cfg, O=None, **kw):
    O = torch.full((Q.shape[0], cfg.nQHeads, cfg.D), 7.0, dtype=Q.dtype, device=DEV) if O is None else O
    cdna4.prefill_packed(Q, K, V, O, cu_d, cfg, Kp, Vp, **kw)
    return O


def verify(args, cfg, dtype, O, what=""):
    Q, K, V, Kp, Vp, cu, _, _ = args
    ref, bound, covered = packed_reference(Q, K, V, cu, cfg.D, cfg.nQHeads // cfg.nKVHeads, dtype, Kp, Vp, cfg.prefix)
    assert bool((O[~covered] == 7.0).all()), "rows of no sequence were written"
    return check(O[covered], ref[covered], bound[covered], what)


LENS = {
    "one": [1], "two_empty": [2, 0, 1], "none": [0, 0], "tile": [64], "edges": [63, 65, 1, 128, 127, 129, 32, 31, 33],
    "gaps": [300, 5, 0, 0, 700], "long": [1500, 3], "equal": [200] * 5, "block": [256, 257, 255],
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", list(LENS))
def test_lengths(name, D, dtype):
    args = make(LENS[name], 4, 2, D, dtype, spare=3, seed=1)
    verify(args, args[-1], dtype, run(*args[:5], *args[6:]), name)


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (16, 2), (40, 8), (12, 12)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(heads, D):
    args = make([100, 1, 37, 260], *heads, D, BF16, seed=2)
    verify(args, args[-1], BF16, run(*args[:5], *args[6:]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [1, 31, 32, 33, 63, 64, 65, 100, 128, 129, 191, 192, 193, 256, 320, 449, 1000])
def test_prefix(prefix, D, dtype):
    args = make([5, 130, 1, 0, 300, 64], 4, 2, D, dtype, prefix=prefix, spare=2, seed=prefix)
    verify(args, args[-1], dtype, run(*args[:5], *args[6:]), f"prefix {prefix}")


@pytest.mark.parametrize("layout", ["fused", "heads", "wide", "plain"])
@pytest.mark.parametrize("prefix", [0, 70])
def test_strides(layout, prefix):
    args = make([90, 0, 200, 33], 8, 4, 128, F16, prefix=prefix, seed=3, layout=layout)
    verify(args, args[-1], F16, run(*args[:5], *args[6:]))
    T = args[0].shape[0]
    O = torch.full((8, T, 128), 7.0, dtype=F16, device=DEV).transpose(0, 1)   # head-major output
    verify(args, args[-1], F16, run(*args[:5], *args[6:], O=O))


@pytest.mark.parametrize("batch", [64, 65, 256, 257, 700])
def test_many_sequences(batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 9, (batch,), generator=g).tolist()
    lens[batch // 2] = 140
    lens[-1] = 131
    args = make(lens, 2, 1, 64, F16, spare=1, seed=batch)
    verify(args, args[-1], F16, run(*args[:5], *args[6:]))


LISTED = {   # calls of two rounds of blocks and more, whose blocks are listed first
    "docs": ([2100, 1, 900, 0, 1300, 77, 4000], 40, 8, 128, BF16, 0),
    "docs_prefix": ([700, 0, 1200, 3], 64, 16, 128, F16, 300),
    "heads_in_turn": ([300, 1, 0, 500, 64, 65] * 4, 20, 10, 64, F16, 0),       # 10 pairs of heads over 8 queues
    "three_heads": ([129] * 350, 3, 1, 64, BF16, 0),
    "one_long": ([9000], 16, 16, 64, BF16, 0),
    "equal": ([64] * 40, 64, 8, 128, F16, 0),
    "most_sequences": ([1, 2, 40] * 682 + [5, 9], 4, 4, 64, F16, 40),          # 2,048
    "more_sequences": ([1, 2, 40] * 683, 4, 4, 64, BF16, 0),                   # 2,049: not listed
    "docs_prefix_listed": ([700, 0, 1200, 300], 64, 16, 128, F16, 300),
    "heads_in_turn_listed": ([300, 1, 0, 500, 64, 65] * 6, 20, 10, 128, F16, 0),
    "three_heads_listed": ([129] * 350, 3, 1, 128, BF16, 0),
    "one_long_listed": ([9000], 16, 16, 128, BF16, 0),
    "most_sequences_listed": ([1, 2, 40] * 682 + [5, 9], 4, 4, 128, F16, 40),  # 2,048
    "more_sequences_128": ([1, 2, 40] * 683, 4, 4, 128, BF16, 0),              # 2,049: not listed
}
# not listed: D = 64, too many sequences, or below two rounds
UNLISTED = {n for n, c in LISTED.items() if c[3] == 64} | {"docs_prefix", "more_sequences_128"}


@pytest.mark.parametrize("name", list(LISTED))
def test_listed_blocks(name):
    lens, HQ, HK, D, dtype, prefix = LISTED[name]
    args = make(lens, HQ, HK, D, dtype, prefix=prefix, spare=2, seed=len(lens))
    need = cdna4.prefill_packed_workspace_size(args[-1])
    assert (need > 0) == (name not in UNLISTED)
    one = run(*args[:5], *args[6:], workspace=None)
    for fill in (0, 255):
        ws = torch.full((need + 16,), fill, dtype=torch.uint8, device=DEV)
        assert torch.equal(one, run(*args[:5], *args[6:], workspace=ws[:need] if need else None))
        assert bool((ws[need:] == fill).all())
    assert torch.equal(one, run(*args[:5], *args[6:]))
    verify(args, args[-1], dtype, one, name)


CUT = {   # calls behind a prefix of 1,024 keys and more with fewer than two rounds of blocks: cut along their keys
    "one_token": ([1], 8, 2, 128, BF16, 2048),
    "few_tokens": ([3, 0, 17, 1], 12, 12, 64, F16, 2049),
    "short_block": ([64], 4, 1, 128, F16, 40000),                     # 32 parts
    "one_head": ([200], 1, 1, 64, BF16, 5000),
    "ragged": ([17, 300, 64, 129, 1], 32, 8, 128, BF16, 4001),
    "more_than_a_round": ([600, 17, 701, 333, 450], 32, 8, 128, F16, 2500),
    "own_longer": ([5000, 20], 8, 2, 64, F16, 2048),
    "heads": ([33] * 9, 10, 5, 128, BF16, 3001),
    "a_round_and_more": ([130] * 40, 16, 4, 64, BF16, 2111),
    "ragged_less": ([17, 60, 64, 40, 1], 32, 8, 128, BF16, 4001),
    "short": ([30, 30], 32, 8, 128, F16, 1025),
    "round_of_half_blocks": ([100] * 11, 32, 8, 128, F16, 2048),
    "own_longer_cut": ([500, 20], 8, 2, 64, F16, 2048),
    "a_round_and_few": ([130] * 39, 16, 4, 64, BF16, 3111),
}
UNCUT = {"ragged", "own_longer"}   # more than half a round of blocks


@pytest.mark.parametrize("name", list(CUT))
def test_cut_blocks(name):
    lens, HQ, HK, D, dtype, prefix = CUT[name]
    args = make(lens, HQ, HK, D, dtype, prefix=prefix, spare=2, seed=len(lens))
    need = cdna4.prefill_packed_workspace_size(args[-1])
    assert (need > 0) == (name not in UNCUT)
    outs = []
    for fill in (0, 255):
        ws = torch.full((need + 16,), fill, dtype=torch.uint8, device=DEV)
        outs.append(run(*args[:5], *args[6:], workspace=ws[:need] if need else None))
        assert bool((ws[need:] == fill).all())
    assert torch.equal(*outs) and torch.equal(outs[0], run(*args[:5], *args[6:]))
    verify(args, args[-1], dtype, outs[0], name)
    verify(args, args[-1], dtype, run(*args[:5], *args[6:], workspace=None), name)


def test_cut_blocks_replayed():
    """Which items are cut, and how, follows the lengths in every replay; wrong lengths stay inside."""
    T, P = 1100, 2600
    Q, K, V, Kp, Vp, _, _, _ = make([T], 32, 8, 128, F16, prefix=P, seed=31)
    cfg = cdna4.PackedPrefillCfg(128, 32, 8, 5, T, 0, P, Kp.shape[1])
    need = cdna4.prefill_packed_workspace_size(cfg)
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device=DEV)
    cu_d = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32, device=DEV)
    O = torch.full((T + 8, 32, 128), 7.0, dtype=F16, device=DEV)
    run(Q, K, V, Kp, Vp, cu_d, cfg, O=O[:T], workspace=ws[:need])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(Q, K, V, Kp, Vp, cu_d, cfg, O=O[:T], workspace=ws[:need])
    for lens in ([1100, 0, 0, 0, 0], [60] * 5, [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], None, [17, 700, 300, 3, 80], [40, 0, 0, 0, 0]):
        cu = cu_of(lens) if lens else [0, T, 0, T, -3, T]
        cu_d.copy_(torch.tensor(cu, dtype=torch.int32))
        O.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((ws[need:] == 255).all()) and bool((O[T:] == 7.0).all())
        if lens:
            assert torch.equal(O[:T], run(Q, K, V, Kp, Vp, cu_d, cfg)), lens
            verify((Q, K, V, Kp, Vp, cu, cu_d, cfg), cfg, F16, O[:T], str(lens))


def test_listed_blocks_replayed():
    """The queues start over in every replay, on other lengths."""
    T = 4200
    Q, K, V, _, _, _, _, cfg0 = make([T], 32, 8, 128, F16, seed=21)
    cfg = cdna4.PackedPrefillCfg(128, 32, 8, 5, T, 0, 0, 0)
    ws = torch.empty(cdna4.prefill_packed_workspace_size(cfg), dtype=torch.uint8, device=DEV)
    cu_d = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32, device=DEV)
    O = torch.full((T, 32, 128), 7.0, dtype=F16, device=DEV)
    run(Q, K, V, None, None, cu_d, cfg, O=O, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(Q, K, V, None, None, cu_d, cfg, O=O, workspace=ws)
    for lens in ([4200, 0, 0, 0, 0], [600] * 5, [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [17, 2000, 900, 3, 80]):
        cu = cu_of(lens)
        cu_d.copy_(torch.tensor(cu, dtype=torch.int32))
        O.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(O, run(Q, K, V, None, None, cu_d, cfg, workspace=None)), lens
        verify((Q, K, V, None, None, cu, cu_d, cfg), cfg, F16, O, str(lens))


def test_workspace_refusals():
    args = make([1900, 1300], 64, 16, 128, F16, seed=22)
    need = cdna4.prefill_packed_workspace_size(args[-1])
    with pytest.raises(cdna4.CDNA4Error):
        run(*args[:5], *args[6:], workspace=torch.empty(need - 1, dtype=torch.uint8, device=DEV))
    for bad in ("none", torch.empty(need, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            run(*args[:5], *args[6:], workspace=bad)


def test_first_row_not_zero():
    args = make([30, 129], 4, 4, 128, BF16, first=11, spare=4, seed=5)
    verify(args, args[-1], BF16, run(*args[:5], *args[6:]))


@pytest.mark.parametrize("scale", [0.0, 8.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_peaked_and_flat(scale, dtype):
    """Scores all equal (scale 0), and scores whose maximum keeps moving (one key takes nearly all weight)."""
    args = make([500, 129], 4, 2, 128, dtype, prefix=97, seed=6, scale=scale)
    verify(args, args[-1], dtype, run(*args[:5], *args[6:]))


def test_large_work():
    """Enough blocks for several rounds of the chip, both main loops of the prefix form."""
    args = make([2100, 1, 900, 1300, 77], 16, 4, 128, BF16, prefix=700, seed=7)
    verify(args, args[-1], BF16, run(*args[:5], *args[6:]))
    args = make([2100, 1, 900, 1300, 77], 16, 4, 64, F16, seed=8)
    verify(args, args[-1], F16, run(*args[:5], *args[6:]))


def test_later_keys_of_any_value():
    """K of a later token, whatever it holds, does not reach the rows before it."""
    lens = [100, 40]
    args = make(lens, 2, 2, 128, F16, seed=9)
    Q, K, V, Kp, Vp, cu, cu_d, cfg = args
    K[50] = float("nan")
    K[60] = float("inf")
    O = run(Q, K, V, Kp, Vp, cu_d, cfg)
    ref, bound, _ = packed_reference(Q, K, V, cu, 128, 1, F16)
    check(O[:50], ref[:50], bound[:50])
    check(O[100:], ref[100:], bound[100:])


def test_lengths_outside_the_tensors_stay_inside():
    """Entries of cu past `total`, negative or decreasing: nothing outside the tensors is read or written."""
    T = 300
    guard = torch.full((T + 200, 4, 64), 7.0, dtype=F16, device=DEV)
    x = torch.randn(T, 4, 64, device=DEV).to(F16)
    for cu in ([0, 100, 5000], [-50, 100, 200], [0, 250, 100, 299], [400, 500, 600], [2 ** 31 - 1, -2 ** 31, 7]):
        cu_d = torch.tensor(cu, dtype=torch.int32, device=DEV)
        cfg = cdna4.PackedPrefillCfg(64, 4, 4, len(cu) - 1, T, 0, 0, 0)
        cdna4.prefill_packed(x, x, x, guard[:T], cu_d, cfg)
        assert bool((guard[T:] == 7.0).all())
        guard[:T] = 7.0
    cu_d = torch.tensor([0, 100, 300], dtype=torch.int32, device=DEV)     # and the next call is right again
    cdna4.prefill_packed(x, x, x, guard[:T], cu_d, cdna4.PackedPrefillCfg(64, 4, 4, 2, T, 200, 0, 0))
    ref, bound, _ = packed_reference(x, x, x, [0, 100, 300], 64, 1, F16)
    check(guard[:T], ref, bound)


def test_wrong_lengths_stay_inside_the_list():
    """Overlapping sequences, which have many times the blocks that the workspace lists: nothing outside it, or outside
    the tensors, is written, and the next call is right."""
    T, n = 4200, 64
    x = torch.randn(T, 8, 128, device=DEV).to(F16)
    guard = torch.full((T + 64, 32, 128), 7.0, dtype=F16, device=DEV)
    q = torch.randn(T, 32, 128, device=DEV).to(F16)
    cfg = cdna4.PackedPrefillCfg(128, 32, 8, n, T, 0, 0, 0)
    need = cdna4.prefill_packed_workspace_size(cfg)
    assert need > 0
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device=DEV)
    for cu in ([0, T] * (n // 2) + [0], [0, T, -5] * 21 + [0, T], [T, 0] * (n // 2) + [2 ** 31 - 1]):
        cu_d = torch.tensor(cu, dtype=torch.int32, device=DEV)
        assert cu_d.numel() == n + 1
        for w in (ws[:need], None):
            cdna4.prefill_packed(q, x, x, guard[:T], cu_d, cfg, workspace=w)
        torch.cuda.synchronize()
        assert bool((ws[need:] == 255).all()) and bool((guard[T:] == 7.0).all())
    cu = cu_of([64] * (n - 1) + [T - 64 * (n - 1)])
    cu_d = torch.tensor(cu, dtype=torch.int32, device=DEV)
    guard[:T] = 7.0
    cdna4.prefill_packed(q, x, x, guard[:T], cu_d, cfg, workspace=ws[:need])
    one = torch.empty_like(q)
    cdna4.prefill_packed(q, x, x, one, cu_d, cfg, workspace=None)
    assert torch.equal(one, guard[:T])
    ref, bound, _ = packed_reference(q, x, x, cu, 128, 4, F16)
    check(one, ref, bound)


def test_equal_lengths_as_the_uniform_call():
    """Sequences of one length: what prefill gives for them, within both calls' bounds."""
    B, S, H, D = 3, 333, 8, 128
    args = make([S] * B, H, H, D, BF16, seed=10, layout="plain")
    Q, K, V, _, _, cu, cu_d, cfg = args
    O = run(Q, K, V, None, None, cu_d, cfg)
    hm = lambda t: t.view(B, S, H, D).transpose(1, 2).contiguous()
    U = torch.empty(B, H, S, D, dtype=BF16, device=DEV)
    cdna4.prefill(hm(Q), hm(K), hm(V), U, cdna4.PrefillCfg(D, S, S, H, H, B, 1))
    _, bound, _ = packed_reference(Q, K, V, cu, D, 1, BF16)
    check(O, U.transpose(1, 2).reshape(B * S, H, D).double(), 2 * bound)


def test_stream_and_overlap():
    """Two calls on two streams at once; neither disturbs the other."""
    a = make([400, 30], 8, 2, 128, BF16, seed=11)
    b = make([77, 500, 1], 8, 8, 64, F16, prefix=40, seed=12)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    Oa = torch.full((a[0].shape[0], 8, 128), 7.0, dtype=BF16, device=DEV)
    Ob = torch.full((b[0].shape[0], 8, 64), 7.0, dtype=F16, device=DEV)
    torch.cuda.synchronize()
    for _ in range(5):
        run(*a[:5], *a[6:], O=Oa, stream=s1)
        run(*b[:5], *b[6:], O=Ob, stream=s2)
    torch.cuda.synchronize()
    verify(a, a[-1], BF16, Oa)
    verify(b, b[-1], F16, Ob)


def test_captured_call_replays_on_other_lengths():
    T = 700
    args = make([T], 4, 2, 128, F16, prefix=50, seed=13)
    Q, K, V, Kp, Vp, _, _, _ = args
    cfg = cdna4.PackedPrefillCfg(128, 4, 2, 4, T, 0, 50, 55)
    cu_d = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=DEV)
    O = torch.full((T, 4, 128), 7.0, dtype=F16, device=DEV)
    run(Q, K, V, Kp, Vp, cu_d, cfg, O=O)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(Q, K, V, Kp, Vp, cu_d, cfg, O=O)
    for lens in ([700, 0, 0, 0], [1, 130, 64, 505], [0, 300, 0, 13], [100, 100, 100, 100]):
        cu = cu_of(lens)
        cu_d.copy_(torch.tensor(cu, dtype=torch.int32))
        O.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(Q, K, V, Kp, Vp, cu_d, cfg)
        assert torch.equal(O, eager)
        verify((Q, K, V, Kp, Vp, cu, cu_d, cfg), cfg, F16, O, str(lens))


def test_nothing_to_do():
    x = torch.zeros(0, 4, 64, dtype=F16, device=DEV)
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    cdna4.prefill_packed(x, x, x, x, cu, cdna4.PackedPrefillCfg(64, 4, 4, 0, 0, 0, 0, 0))
