"""cdna4.beam_select against scores in 64 bits, and cdna4.paged_reorder against copies made by indexing."""
import math

import pytest
import torch

import cdna4
from paged_util import Paged
from serving_util import DEV

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def reference(logits, cum, beams, n, done=None, eos=-1):
    """Scores in 64 bits, all candidates of a group sorted, equal ones by place."""
    M, V = logits.shape
    x = logits.double().nan_to_num(nan=-math.inf, posinf=torch.finfo(F32).max, neginf=-math.inf)
    top = x.amax(1, keepdim=True)
    alive = (top[:, 0] > -math.inf) & torch.isfinite(cum)
    x = x - torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = x - x.exp().sum(1, keepdim=True).log().clamp(min=0) + cum.double()[:, None]
    x[~alive] = -math.inf
    if done is not None:
        ended = done != 0
        x[ended] = -math.inf
        x[ended, eos] = torch.where(torch.isfinite(cum[ended]), cum[ended].double(), torch.full_like(cum[ended].double(), -math.inf))
    x = x.view(M // beams, beams * V)
    score, at = torch.sort(x, dim=1, descending=True, stable=True)
    if score.shape[1] < n:
        pad = n - score.shape[1]
        score = torch.nn.functional.pad(score, (0, pad), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, pad))
    score, at = score[:, :n], at[:, :n]
    none = score == -math.inf
    first = torch.arange(M // beams, device=logits.device)[:, None] * beams
    return score, torch.where(none, -1, first + at // V).int(), torch.where(none, -1, at % V).int()


def verify(logits, cum, beams, n=None, **kw):
    got = cdna4.beam_select(logits, cum, beams, n, **kw)
    want = reference(logits, cum, beams, n or beams, kw.get("done"), kw.get("eos", -1))
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    # a row's sum of exponentials: V / 64 additions of a lane and 16 roundings more, each 2^-24; then the score's own rounding
    off = (logits.shape[1] / 64 + 16) * 2.0 ** -24
    fine = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0]), fine)
    d = (got[0].double() - want[0]).abs()[fine]
    assert bool((d <= off + 2.0 ** -23 * want[0][fine].abs()).all())
    return got


def make(G, beams, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(G * beams, V, device=DEV, generator=g) * spread).to(dtype), -20 * torch.rand(G * beams, device=DEV, generator=g)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4097, 32000, 100003])
def test_vocabularies(V, dtype):
    """16-bit logits have many ties; the vocabulary may be smaller than the number wanted."""
    x, cum = make(3, 4, V, dtype, seed=V)
    verify(x, cum, 4, 8)


@pytest.mark.parametrize("beams,n", [(1, 1), (1, 64), (2, 3), (5, 10), (8, 8), (16, 32), (33, 40), (64, 64)])
@pytest.mark.parametrize("G", [1, 3])
def test_beams(G, beams, n):
    x, cum = make(G, beams, 2500, BF16, seed=beams)
    verify(x, cum, beams, n)


@pytest.mark.parametrize("G", [40, 300])
def test_many_groups(G):
    x, cum = make(G, 4, 3000, F16, seed=G)
    verify(x, cum, 4, 8)


def test_ties_go_to_the_lowest_place():
    x = torch.zeros(8, 5000, device=DEV)
    cum = torch.zeros(8, device=DEV)
    got = verify(x, cum, 4, 16)
    assert got[2][0].tolist() == list(range(16)) and bool((got[1][0] == 0).all()) and bool((got[1][1] == 4).all())
    x[:, 4990:] = 1.0                                        # ten best of each row, at its end
    got = verify(x, cum, 4, 16)
    assert got[2][0].tolist() == list(range(4990, 5000)) + list(range(4990, 4996)) and got[1][0].tolist() == [0] * 10 + [1] * 6
    ramp = torch.arange(5000, device=DEV).float().repeat(8, 1) / 100
    verify(ramp, cum, 4, 16)                                 # every chunk better than the one before
    verify(-ramp, cum, 4, 16)
    verify(ramp.half(), cum, 4, 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [2048, 5001, 40000, 100003])
def test_equal_logits_over_many_steps(V, dtype):
    """Rows flat, flat but for some late ones, flat in stretches, of the lowest value but for a few, zeros of both signs, and rising."""
    x, cum = torch.zeros(8, V, dtype=dtype, device=DEV), torch.zeros(8, device=DEV)
    low = torch.finfo(dtype).min
    x[1, -3:] = 0.5
    x[2] = (torch.arange(V, device=DEV) // 500 % 3).to(dtype)
    x[3] = low
    x[3, [7, V // 2, V - 1]] = torch.tensor([1.0, 3.0, 2.0], device=DEV).to(dtype)
    x[4, ::2] = -0.0
    x[5] = (torch.arange(V, device=DEV) // 64).to(dtype)
    x[6] = -x[5]
    x[7] = low
    for n in (1, 4, 16, 64):
        verify(x, cum, 1, n)
        verify(x, cum, 4, n)


def test_time_of_equal_logits():
    """A mask of a finite value over most of a vocabulary takes a few times as long as random logits: 1.7 times; 30 where every equal logit
    is inserted."""
    rows, V, beams, n = 256, 100003, 8, 16
    x, cum = make(rows // beams, beams, V, BF16, seed=n)
    flat = torch.full_like(x, torch.finfo(BF16).min)
    flat[:, :5] = x[:, :5]
    ws = torch.empty(cdna4.beam_select_workspace_size(rows, V, beams, n), dtype=torch.uint8, device=DEV)
    best = []
    for y in (x, flat):
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(20):
                out = cdna4.beam_select(y, cum, beams, n, workspace=ws)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        best.append(min(times))
    assert best[1] < 8 * best[0], best


def test_order_within_a_row_is_that_of_its_logits():
    """Also where a large cum leaves nothing of their differences in a score."""
    x, _ = make(1, 2, 5000, F32, seed=9)
    x[1] = x[0]
    for c in (-1e9, -1e20, 1e30):
        s, p, t = cdna4.beam_select(x, torch.full((2,), c, device=DEV), 1, 8)
        assert torch.equal(t.long(), x.topk(8, dim=1).indices) and bool((s == c).all())
    s, p, t = cdna4.beam_select(x, torch.full((2,), -1e20, device=DEV), 2, 8)   # equal scores: the lowest row's
    assert bool((p == 0).all()) and torch.equal(t[0].long(), x[0].topk(8).indices)


def test_masks_and_values_that_are_not_finite():
    x, cum = make(4, 4, 3000, F32, seed=1)
    x[0, 5:] = -math.inf                                     # few tokens allowed
    x[1] = -math.inf                                         # none
    x[2, ::2] = float("nan")
    x[3] = torch.finfo(F32).min                              # a mask of the type's lowest value over everything
    x[4:8] = -math.inf                                       # a group without any
    x[8, 17] = math.inf
    x[9, 3], x[9, 700] = math.inf, math.inf
    x[10] = torch.finfo(F32).min
    x[10, 1234] = 2.0
    got = verify(x, cum, 4, 8)
    assert bool((got[1][1] == -1).all()) and bool((got[2][1] == -1).all()) and bool((got[0][1] == -math.inf).all())
    h = x.clone().clamp(-65504, 65504).half()
    h[0, 5:] = -math.inf
    verify(h, cum, 4, 8)
    cum[0], cum[5], cum[9] = -math.inf, math.inf, float("nan")   # unused beams
    verify(x, cum, 4, 8)
    first = torch.tensor([0.0, -math.inf, -math.inf, -math.inf] * 4, device=DEV)   # a search's first step
    got = verify(make(4, 4, 3000, F32, seed=2)[0], first, 4, 4)
    assert torch.equal(got[1][:, 0], torch.arange(0, 16, 4, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [4095, 4096, 4100, 5003, 40000])
def test_ranges_of_a_row(V, dtype):
    """Rows cut into ranges that share what they know: best logits all in one range, ranges of NaN or -inf, +inf in some, ends."""
    x, cum = make(3, 6, V, dtype, seed=V)
    q = V // 4
    x[0, :q] += 40                                           # all best ones in the first range, in the last, at both ends
    x[1, -q:] += 40
    x[2, 0], x[2, -1] = 60.0, 60.0
    x[3, :q] = float("nan")                                  # a range without any
    x[4, q:] = float("nan")                                  # few left
    x[5, q:2 * q] = -math.inf
    x[6, 2 * q:] = -math.inf
    x[7, 5::1000] = math.inf
    x[8, 3 * q + 5] = math.inf
    x[9] = -math.inf
    x[9, V - 3] = 1.0
    x[10, 1:] = float("nan")
    x[11] = 2.0                                              # equal everywhere
    x[12] = torch.linspace(-5, 5, V, device=DEV).to(dtype)   # the best ones come last
    x[13] = torch.linspace(5, -5, V, device=DEV).to(dtype)
    for n in (1, 5, 12, 64):
        verify(x, cum, 6, n)


@pytest.mark.parametrize("beams,n,V", [(64, 64, 9001), (1, 64, 50001), (16, 3, 6000), (17, 64, 5000)])
def test_many_wanted(beams, n, V):
    x, cum = make(2, beams, V, BF16, seed=n)
    cum[1] = -math.inf
    verify(x, cum, beams, n)
    cum[:beams - 1] = -math.inf                              # one row has them all
    verify(x, cum, beams, n)


def test_beams_that_have_ended():
    x, cum = make(3, 4, 2000, F16, seed=3)
    done = torch.tensor([0, 1, 0, 5, 1, 1, 1, 1, 0, 0, 0, 0], dtype=torch.int32, device=DEV)
    cum[1], cum[5] = 3.0, -math.inf                          # the best of its group; one that never was
    x[3] = float("nan")
    got = verify(x, cum, 4, 8, done=done, eos=7)
    assert int(got[1][0, 0]) == 1 and int(got[2][0, 0]) == 7 and float(got[0][0, 0]) == 3.0
    assert got[1][1].tolist()[3:] == [-1] * 5                # three ended beams, five empty places


def test_rows_apart_and_outputs_given():
    wide, cum = make(2, 3, 5001, BF16, seed=4)
    x = wide[:, 3:4500]                                      # odd offset, odd length
    assert x.stride(0) == 5001
    out = tuple(torch.zeros(2, 6, dtype=d, device=DEV) for d in (F32, torch.int32, torch.int32))
    got = verify(x, cum, 3, 6, out=out)
    assert got is out
    need = cdna4.beam_select_workspace_size(6, 4497, 3, 6)
    for fill in (0, 255):
        ws = torch.full((need + 64,), fill, dtype=torch.uint8, device=DEV)
        again = cdna4.beam_select(x, cum, 3, 6, workspace=ws[:need])
        assert all(torch.equal(a, b) for a, b in zip(got, again)) and bool((ws[need:] == fill).all())
    with pytest.raises(cdna4.CDNA4Error):
        cdna4.beam_select(x, cum, 3, 6, workspace=ws[:need - 1])
    for bad in (dict(workspace=None), dict(workspace="none"), dict(out=tuple(t[:1] for t in out)), dict(done=cum)):
        with pytest.raises(ValueError):
            cdna4.beam_select(x, cum, 3, 6, **bad)
    with pytest.raises(ValueError):
        cdna4.beam_select(x, cum, 4)                         # six rows
    with pytest.raises(cdna4.CDNA4Error):
        cdna4.beam_select(x, cum, 3, 65)


@pytest.mark.parametrize("beams,n,V", [(1, 3, 400001), (2, 2, 270000), (2, 40, 300000)])
def test_more_ranges_than_a_load_of_their_keys(beams, n, V):
    """Over 256 ranges to a row: the best of some lie behind the first keys read."""
    x, cum = make(1, beams, V, BF16, seed=V)
    verify(x, cum, beams, n)
    x[:, V - 5:] = torch.arange(20, 25, device=DEV).to(BF16)  # rising to the end
    verify(x, cum, beams, n)


def test_scores_in_the_place_of_cum():
    for G, beams, V in ((1, 4, 32000), (33, 7, 3001)):
        x, cum = make(G, beams, V, F16, seed=V)
        want = cdna4.beam_select(x, cum.clone(), beams)
        out = (cum, torch.empty(G, beams, dtype=torch.int32, device=DEV), torch.empty(G, beams, dtype=torch.int32, device=DEV))
        cdna4.beam_select(x, cum, beams, out=out)
        assert torch.equal(cum.view(G, beams), want[0]) and torch.equal(out[1], want[1]) and torch.equal(out[2], want[2])


def test_scores_in_the_place_of_cum_of_another_number_are_refused():
    for n in (2, 6):
        x, cum = make(3, 4, 3000, F16, seed=n)
        room = torch.zeros(max(12, 3 * n), device=DEV)       # both at one address, each long enough
        room[:12] = cum
        out = (room, torch.empty(3, n, dtype=torch.int32, device=DEV), torch.empty(3, n, dtype=torch.int32, device=DEV))
        with pytest.raises(cdna4.CDNA4Error):
            cdna4.beam_select(x, room, 4, n, out=out)
        assert torch.equal(room[:12], cum)


def test_logits_past_32_bit_offsets():
    V = 1 << 20
    x = torch.full((2100, V), -math.inf, dtype=F16, device=DEV)   # 4.4 GB
    x[:, 5] = 1.0
    x[2099, V - 1], x[2099, V - 2] = 3.0, 2.0
    cum = torch.zeros(2100, device=DEV)
    s, p, t = cdna4.beam_select(x, cum, 1, 2)
    assert t[2099].tolist() == [V - 1, V - 2] and p[2099].tolist() == [2099, 2099]
    assert bool((t[:2099, 0] == 5).all()) and bool((t[:2099, 1] == -1).all()) and bool((s[:2099, 0] == 0).all())


def test_captured_and_on_another_stream():
    x, cum = make(4, 4, 8000, BF16, seed=5)
    out = tuple(torch.zeros(4, 8, dtype=d, device=DEV) for d in (F32, torch.int32, torch.int32))
    ws = torch.empty(cdna4.beam_select_workspace_size(16, 8000, 4, 8), dtype=torch.uint8, device=DEV)
    cdna4.beam_select(x, cum, 4, 8, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cdna4.beam_select(x, cum, 4, 8, out=out, workspace=ws)
    for i in range(4):
        y, c = make(4, 4, 8000, BF16, seed=6 + i)
        x.copy_(y), cum.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        eager = cdna4.beam_select(x, cum, 4, 8, stream=s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        verify(x, cum, 4, 8)


# ---- reorder ----------------------------------------------------------------------------------------

def reorder_reference(parents, tables, lens, fresh, K, V, page, pages, most, fmt, D):
    """tables_out, lens_out and pools after the copies, row by row."""
    t = torch.full((len(parents), tables.shape[1]), -1, dtype=torch.int32)
    l = torch.zeros(len(parents), dtype=torch.int32)
    K0, V0, K, V = K, V, K.clone(), V.clone()
    for i, p in enumerate(parents):
        if not 0 <= p < len(lens):
            continue
        n = min(max(lens[p], 0), most)
        t[i], l[i] = tables[p], n
        if n % page == 0:
            continue
        src = int(tables[p, n // page])
        t[i, n // page] = fresh[i]
        if 0 <= src < pages and 0 <= fresh[i] < pages:
            r = n % page
            for pool, old in ((K, K0), (V, V0)):
                if fmt == "mxfp4":
                    c = page * D // 2
                    pool[..., fresh[i], :, :r * D // 2] = old[..., src, :, :r * D // 2]
                    pool[..., fresh[i], :, c:c + r * D // 32] = old[..., src, :, c:c + r * D // 32]
                else:
                    pool[..., fresh[i], :, :r, :] = old[..., src, :, :r, :]
    return t, l, K, V


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("layers", [0, 1, 3])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 256), (128, 32), (128, 64)])
def test_reorder(D, page, layers, fmt):
    lens = [0, 1, 15, 16, 17, 100, 255, 256, 300]
    rows = len(lens)
    p = Paged(lens, 3, D, F16, page, fmt, seed=D, spare=rows + 4)
    g = torch.Generator(device=DEV)
    g.manual_seed(page)
    shape = ((layers,) if layers else ()) + cdna4.paged_pool_shape(p.cache)
    if fmt == "mxfp4":
        K, V = (torch.randint(0, 256, shape, device=DEV, generator=g, dtype=torch.int32).to(torch.uint8) for _ in range(2))
    else:
        K, V = (torch.randn(*shape, device=DEV, generator=g).half() for _ in range(2))
    parents = [8, 8, 5, 0, 4, -1, 6, 1, 2, 9, 8]             # more rows than before, two of them unused
    fresh = p.free[:len(parents)]
    fresh[6] = int(p.tables[6, 255 // page])                 # the parent's own page: its only successor
    want = reorder_reference(parents, p.tables.cpu(), lens, fresh, K, V, page, p.cache.pages, p.cache.max_pages * page, fmt, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    to, lo = torch.full((len(parents), p.tables.shape[1]), 99, dtype=torch.int32, device=DEV), i32([99] * len(parents))
    cdna4.paged_reorder(i32(parents), p.tables, p.lens, i32(fresh), to, lo, K, V, p.cache)
    assert torch.equal(to.cpu(), want[0]) and torch.equal(lo.cpu(), want[1]) and torch.equal(K, want[2]) and torch.equal(V, want[3])


def test_reorder_of_bad_pages_and_lengths():
    """Pages outside the pool are named and not touched; lengths are cut to the table."""
    p = Paged([20, 40, 30], 2, 64, F16, 16, "16", spare=6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    p.tables[1, 2] = 10 ** 6
    fresh = [-7, p.free[0], 10 ** 7]
    lens = [20, 40, 2 ** 31 - 1]
    K0, V0 = p.K.clone(), p.V.clone()
    to, lo = torch.zeros_like(p.tables), torch.zeros_like(p.lens)
    cdna4.paged_reorder(i32([0, 1, 2]), p.tables, i32(lens), i32(fresh), to, lo, p.K, p.V, p.cache)
    t = p.tables.clone()
    t[0, 1], t[1, 2] = -7, p.free[0]                          # the third is cut to whole pages
    assert torch.equal(to, t) and lo.tolist() == [20, 40, p.cache.max_pages * 16]
    bits = lambda x: x.view(torch.int16)
    assert torch.equal(bits(p.K), bits(K0)) and torch.equal(bits(p.V), bits(V0))
    with pytest.raises(cdna4.CDNA4Error):
        cdna4.paged_reorder(i32([0, 1, 2]), p.tables, p.lens, i32(fresh), p.tables, lo, p.K, p.V, p.cache)
    with pytest.raises(ValueError):
        cdna4.paged_reorder(i32([0, 1, 2]), p.tables, p.lens, i32([1]), to, lo, p.K, p.V, p.cache)
