"""cdna4.decode_paged against a 64-bit reference: lengths from no key to many shares, page sizes, both formats, head layouts,
several queries, lengths and tables read on the device. `form`: "whole", a table of few pages, a workgroup per item; "shares", one
long enough for equal shares of all keys, whatever the lengths."""
import pytest
import torch

import cdna4
from paged_util import Paged, attend_two_terms, decode_reference
from serving_util import DEV, check

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


FORMS = pytest.mark.parametrize("form", ["whole", "shares"])


def make(lens, HQ, HK, D, dtype, page=16, fmt="16", nq=1, seed=0, scale=1.0, form="whole"):
    p = Paged(lens, HK, D, dtype, page, fmt, seed, room=min(2, 256 // page) if form == "whole" else 4096 // page)
    q = (torch.randn(len(lens), nq, HQ, D, device=DEV, generator=p.g) * scale).to(dtype)
    cfg = cdna4.PagedDecodeCfg(HQ, len(lens), nq)
    if max(lens, default=0) <= 700 and len(lens) <= 130:     # `room` decides there
        assert (cdna4.decode_paged_plan(p.cache, cfg).workspace == 0) == (form == "whole")
    return p, q, cfg


def run(p, q, cfg, o=None, tables=None, lens=None, **kw):
    o = torch.full_like(q, 7.0) if o is None else o
    cdna4.decode_paged(q, p.K, p.V, p.tables if tables is None else tables, p.lens if lens is None else lens, o, p.cache, cfg, **kw)
    return o


def verify(p, q, o, what=""):
    return check(o, *decode_reference(q, p.k, p.v, q.dtype), what)


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_lengths(page, D, dtype, fmt, form):
    """Pages that end inside a chunk, at it and past it; rows behind the last one are NaN."""
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 64, 65, 100, 255, 256, 257, 300, 700]
    p, q, cfg = make(lens, 8, 2, D, dtype, page, fmt, seed=page, form=form)
    o = run(p, q, cfg)
    verify(p, q, o, f"page {page}")
    assert bool((o[0] == 0).all())


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (16, 2), (40, 8), (12, 12), (20, 1), (33, 1), (64, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(heads, D, fmt, form):
    p, q, cfg = make([70, 0, 129], *heads, D, F16, 32, fmt, seed=heads[0], form=form)
    verify(p, q, run(p, q, cfg))


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("nq", [2, 3, 5, 8, 16])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (20, 2)])
def test_several_queries(heads, nq, fmt, form):
    """Sequences shorter than the queries leave the first ones nothing to see: zeros."""
    lens = [0, 1, nq - 1, nq, 31, 32, 33, 40, 95, 300]
    p, q, cfg = make(lens, *heads, 64 if nq == 3 else 128, BF16 if nq == 2 else F16, 16, fmt, nq, seed=nq, form=form)
    # a query whose row sees nothing gets 0 times the sequence's values, which are finite here
    o = run(p, q, cfg)
    verify(p, q, o)
    for b, n in enumerate(lens):
        assert bool((o[b, :max(nq - n, 0)] == 0).all())


@FORMS
@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 130, 1000, 4099])
def test_batches(B, form):
    """More sequences than a wave's lanes, and than 64 lanes of 64, most of them empty."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g)
    lens[torch.rand(B, generator=g) < (0.3 if B < 1000 else 0.9)] = 0
    lens = lens.tolist()
    p, q, cfg = make(lens, 4, 1, 64, BF16, 16, seed=B, form=form)
    verify(p, q, run(p, q, cfg))


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_long(fmt):
    """Shares of many chunks, items cut into many shares, page ids past a wave's 64."""
    lens = [40000, 17, 9000, 0, 2500, 33]
    for D, dtype, page in ((128, BF16, 16), (64, F16, 64)):
        p, q, cfg = make(lens, 8, 2, D, dtype, page, fmt, seed=2)
        verify(p, q, run(p, q, cfg))


def test_one_long_among_short():
    lens = [30] * 100 + [20000] + [50] * 27
    p, q, cfg = make(lens, 4, 2, 64, F16, 32, seed=3)
    verify(p, q, run(p, q, cfg))


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("scale", [0.0, 8.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_peaked_and_flat(scale, dtype, fmt, form):
    p, q, cfg = make([300, 0, 64], 8, 2, 128, dtype, 32, fmt, seed=4, scale=scale, form=form)
    verify(p, q, run(p, q, cfg))


@pytest.mark.parametrize("rows", [96, 4096])
def test_lengths_are_cut_and_tables_clamped(rows):
    """Lengths outside the table's rows are cut to them; entries outside the pool read some page of it and touch no other sequence."""
    lens = [rows + 4, 0, rows, 60]
    p, q, cfg = make(lens, 4, 2, 64, F16, 16, seed=5)
    p.cache.max_pages, p.cache.table_stride = rows // 16, p.tables.shape[1]
    o = run(p, q, cfg, lens=torch.tensor([2 ** 31 - 1, -2 ** 31, rows + 1, 60], dtype=torch.int32, device=DEV))
    p.k, p.v = [x[:, :rows] for x in p.k], [x[:, :rows] for x in p.v]
    verify(p, q, o)
    t = p.tables.clone()
    t[3, 1], t[3, 2] = -5, 2 ** 30
    o2 = run(p, q, cfg, tables=t, lens=torch.tensor([rows + 4, 0, rows + 4, 60], dtype=torch.int32, device=DEV))
    assert torch.equal(o2[:3], o[:3])


@FORMS
def test_shared_pages_equal_copies(form):
    """Two tables naming the same pages give the same bits as each alone."""
    p, q, cfg = make([200], 8, 2, 128, BF16, 32, seed=6, form=form)
    t, l = p.tables.repeat(3, 1), p.lens.repeat(3)
    q3 = q.repeat(3, 1, 1, 1)
    o = torch.empty_like(q3)
    cdna4.decode_paged(q3, p.K, p.V, t, l, o, p.cache, cdna4.PagedDecodeCfg(8, 3, 1))
    verify(p, q, o[:1])
    ref, bound = decode_reference(q, p.k, p.v, BF16)
    for i in (1, 2):
        check(o[i:i + 1], ref, bound)


def test_as_decode_of_a_contiguous_cache():
    lens = [777] * 3
    p, q, cfg = make(lens, 8, 2, 128, F16, 64, seed=7)
    o = run(p, q, cfg)
    u = torch.empty(3, 8, 128, dtype=F16, device=DEV)
    K, V = torch.stack(p.k).to(F16), torch.stack(p.v).to(F16)
    cdna4.decode(q[:, 0].contiguous(), K, V, u, cdna4.DecodeCfg(128, 777, 8, 2, 3, 0))
    _, bound = decode_reference(q, p.k, p.v, F16)
    check(o[:, 0], u.double(), 2 * bound[:, 0])


@FORMS
def test_masked_keys_that_are_not_finite(form):
    """K rows that some queries must not see may hold anything; a V that is not finite stays with the queries that see it and those of up
    to nq - 1 tokens before it."""
    p, q, cfg = make([50, 70], 4, 2, 64, F16, 16, nq=3, seed=8, form=form)
    ref, bound = decode_reference(q, p.k, p.v, F16)
    last = int(p.tables[0, 49 // 16])
    p.K[last, :, 49 % 16] = float("nan")                     # row 49: queries 0 and 1 must not see it
    o = run(p, q, cfg)
    check(o[0, :2], ref[0, :2], bound[0, :2])
    check(o[1], ref[1], bound[1])
    assert bool(o[0, 2].isnan().all())


def test_workspace_contents_do_not_matter():
    p, q, cfg = make([40, 0, 2000], 8, 2, 128, F16, 32, seed=9)   # equal shares
    need = cdna4.decode_paged_workspace_size(p.cache, cfg)
    a = run(p, q, cfg)
    for fill in (0, 255):
        ws = torch.full((need + 64,), fill, dtype=torch.uint8, device=DEV)
        assert torch.equal(a, run(p, q, cfg, workspace=ws[:need]))
        assert bool((ws[need:] == fill).all())
    with pytest.raises(cdna4.CDNA4Error):
        run(p, q, cfg, workspace=ws[:need - 1])
    for bad in (None, "none"):
        with pytest.raises(ValueError):
            run(p, q, cfg, workspace=bad)
    with pytest.raises(ValueError):
        run(p, q, cfg, tables=p.tables[:2])
    with pytest.raises(ValueError):
        run(p, q.to(BF16), cfg)


def test_two_streams_at_once():
    a, b = make([400, 30, 0], 8, 2, 128, BF16, 16, seed=10, form="shares"), make([77, 500], 12, 12, 64, F16, 32, "mxfp4", seed=11)
    oa, ob = torch.empty_like(a[1]), torch.empty_like(b[1])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        run(*a, o=oa, stream=s1)
        run(*b, o=ob, stream=s2)
    torch.cuda.synchronize()
    verify(a[0], a[1], oa)
    verify(b[0], b[1], ob)


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_captured_call_replays_on_other_lengths(fmt, form):
    p, q, cfg = make([600] * 4, 8, 2, 128, F16, 32, fmt, seed=12, form=form)
    full_k, full_v = p.k, p.v
    ws = torch.empty(cdna4.decode_paged_workspace_size(p.cache, cfg), dtype=torch.uint8, device=DEV)
    o = torch.empty_like(q)
    run(p, q, cfg, o=o, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(p, q, cfg, o=o, workspace=ws)
    for lens in ([0, 0, 0, 0], [1, 600, 33, 64], [599, 2, 0, 300], [600] * 4):
        p.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, run(p, q, cfg))
        p.k, p.v = [x[:, :n] for x, n in zip(full_k, lens)], [x[:, :n] for x, n in zip(full_v, lens)]
        verify(p, q, o, str(lens))


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_pools_past_32_bit_offsets(fmt, form):
    """The rows of interest lie in the last pages of a pool of more than 4 GiB."""
    HK, D, page = 8, 128, 256
    pages = 2 ** 32 // (HK * page * (256 if fmt == "16" else 68)) + 40
    p, q, cfg = make([900, 300], 16, HK, D, F16, page, fmt, seed=13, form=form)
    small = p.cache.pages
    for name in ("K", "V"):
        old = getattr(p, name)
        pool = torch.zeros((pages,) + tuple(old.shape[1:]), dtype=old.dtype, device=DEV)
        pool[pages - small:] = old
        setattr(p, name, pool)
    p.cache.pages = pages
    p.tables = torch.where(p.tables >= 0, p.tables + (pages - small), p.tables)
    verify(p, q, run(p, q, cfg))


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("nq", [1, 5])
@pytest.mark.parametrize("D, n", [(64, 60), (64, 120), (64, 250), (64, 2040), (128, 60), (128, 120), (128, 250), (128, 1020)])
def test_waves_per_item(D, n, nq, fmt):
    """One to eight waves per item; the last has 20 heads x 5 queries, several row blocks."""
    lens = [n, 0, n // 2 + 1, 1, n - 1]
    p, q, cfg = make(lens, 20, 2, D, BF16, 16, fmt, nq, seed=n)
    p.cache.max_pages, p.cache.table_stride = (n + 15) // 16, p.tables.shape[1]
    plan = cdna4.decode_paged_plan(p.cache, cfg)
    chunks = (n + 31) // 32
    assert plan.workspace == 0 and plan.waves == min(chunks, 8 if D == 64 or (fmt != "16" and nq == 1) else 4)
    ws = torch.empty(0, dtype=torch.uint8, device=DEV)
    verify(p, q, run(p, q, cfg, workspace=ws))


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("D", [64, 128])
def test_one_wave_per_item(D, fmt):
    """More sequences than the chip holds waves: whole items to a wave, several rounds of them."""
    lens = [(7 * i) % 65 for i in range(5000)]
    p, q, cfg = make(lens, 2, 1, D, F16, 64, fmt, seed=14)
    p.cache.max_pages, p.cache.table_stride = 1, p.tables.shape[1]
    assert cdna4.decode_paged_plan(p.cache, cfg).waves == 1 and cdna4.decode_paged_plan(p.cache, cfg).grid == 5000
    verify(p, q, run(p, q, cfg))


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("nq", [1, 5])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_outputs_are_off_by_their_own_rounding(D, dtype, nq, fmt, form):
    """Weights of one 16-bit term would move an output as far as its rounding does. Small scores, so that the bound's part for them is
    far below that; as many keys as a wave's and several waves' chunks."""
    p, q, cfg = make([300, 0, 33, 250, 120], 20, 2, D, dtype, 16, fmt, nq, seed=21, form=form)
    q /= 64
    o = run(p, q, cfg)
    check(o, *decode_reference(q, p.k, p.v, dtype, attend_two_terms))
    full = torch.randn(q.shape, device=DEV, generator=p.g).to(dtype)
    check(run(p, full, cfg), *decode_reference(full, p.k, p.v, dtype, attend_two_terms))


@FORMS
@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("B", [131, 1000, 4099])
def test_form_of_large_batches(B, fmt, form):
    """Short tables take one launch at any batch, long ones equal shares, in both formats."""
    lens = [(37 * i) % 91 if i % 3 else 0 for i in range(B)]
    p, q, cfg = make(lens, 4, 1, 64, F16, 16, fmt, seed=B, form=form)
    assert (cdna4.decode_paged_plan(p.cache, cfg).workspace == 0) == (form == "whole")
    verify(p, q, run(p, q, cfg))


@pytest.mark.parametrize("D,B,n", [(128, 600, 1280), (128, 600, 2048), (64, 800, 1600)])
def test_rounds_of_several_waves_per_item(D, B, n):
    """MXFP4 in one launch with more waves than the chip holds at once, five to eight chunks in each."""
    lens = [n if i % 50 == 0 else (97 * i) % (n + 1) if i % 4 else i % 3 for i in range(B)]
    p, q, cfg = make(lens, 8, 2, D, F16, 256, "mxfp4", seed=22)
    p.cache.max_pages, p.cache.table_stride = (n + 255) // 256, p.tables.shape[1]
    plan = cdna4.decode_paged_plan(p.cache, cfg)
    assert plan.workspace == 0 and plan.waves == 8 and 5 <= p.cache.max_pages * 256 // 32 / 8 <= 8
    assert plan.grid * plan.waves > 2 * torch.cuda.get_device_properties(DEV).multi_processor_count * 16
    o = run(p, q, cfg)
    verify(p, q, o)
    assert torch.equal(o, run(p, q, cfg))


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_sequences_alike_give_the_same_bits(fmt):
    """A workgroup per item knows nothing of the others."""
    p, q, cfg = make([200], 8, 2, 128, BF16, 32, fmt, seed=23)
    q5, o = q.repeat(5, 1, 1, 1), torch.empty(5, 1, 8, 128, dtype=BF16, device=DEV)
    five = cdna4.PagedDecodeCfg(8, 5, 1)
    assert cdna4.decode_paged_plan(p.cache, five).workspace == 0
    cdna4.decode_paged(q5, p.K, p.V, p.tables.repeat(5, 1), p.lens.repeat(5), o, p.cache, five)
    assert all(torch.equal(o[:1], o[i:i + 1]) for i in range(1, 5))
    verify(p, q, o[:1])
