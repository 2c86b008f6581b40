"""cdna4.rope_append_paged against 64-bit references: what the pools, q_out, k_out and v_out hold, and that nothing else changes."""
import pytest
import torch

import cdna4
from paged_util import append_reference, quantise, unpack, values
from serving_util import DEV, unit

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
EPS = 1e-6


class Call:
    """Tokens of sequences at given first positions, in one projection's output; pools, outputs and tables with room around them."""

    def __init__(self, lens, first, HQ, HK, D, dtype, page, fmt, norm=True, rope=True, seed=0, padding=0, later=0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
        self.HQ, self.HK, self.D, self.page, self.fmt, self.dtype = HQ, HK, D, page, fmt, dtype
        T = sum(lens) + padding
        ends = [f + n for f, n in zip(first, lens)]
        need = [(e + later + page - 1) // page for e in ends]   # room for `later` more tokens
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
        seqs, pos = [], []
        for b, n in enumerate(lens):
            self.tables[b, :need[b]] = torch.tensor(order[:need[b]], dtype=torch.int32)
            order = order[need[b]:]
            seqs += [b] * n
            pos += range(first[b], first[b] + n)
        perm = torch.randperm(T, generator=torch.Generator().manual_seed(seed + 1))      # tokens in any order
        self.seqs = torch.tensor(seqs + [-1] * padding, dtype=torch.int32)[perm].to(DEV)
        self.positions = torch.tensor(pos + [0] * padding, dtype=torch.int32)[perm].to(DEV)
        self.tables = self.tables.to(DEV)
        self.T = T
        qkv = rnd(T, HQ + 2 * HK, D).to(dtype)
        self.q, self.k, self.v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
        self.cache = cdna4.PagedCache(D, HK, page, pages, cdna4.KV_MXFP4 if fmt == "mxfp4" else cdna4.KV_16BIT, self.tables.shape[1])
        shape = cdna4.paged_pool_shape(self.cache)
        if fmt == "mxfp4":
            self.K, self.V = (torch.randint(0, 256, shape, device=DEV, generator=g, dtype=torch.int32).to(torch.uint8) for _ in range(2))
        else:
            self.K, self.V = rnd(*shape).to(dtype), rnd(*shape).to(dtype)
        self.wq, self.wk = ((1 + 0.2 * rnd(D)).to(dtype) if norm else None for _ in range(2))
        self.cos = self.sin = None
        if rope:
            self.cos, self.sin = cdna4.rope_table_f32(0, max(ends + [1]) + later, D, 10000.0, device=DEV)
        self.q_out = torch.full((T, HQ, D), 7.0, dtype=dtype, device=DEV)
        self.k_out, self.v_out = (torch.full((T, HK, D), 7.0, dtype=dtype, device=DEV) for _ in range(2))

    def run(self, **kw):
        args = dict(seqs=self.seqs, cos=self.cos, sin=self.sin, q_norm=self.wq, k_norm=self.wk, eps=EPS, k_out=self.k_out, v_out=self.v_out)
        args.update(kw)
        return cdna4.rope_append_paged(self.q, self.k, self.v, self.K, self.V, self.tables, self.positions, self.cache, self.q_out, **args)

    def live(self):
        """Tokens that are written, their positions, pages and rows."""
        t = (self.seqs >= 0).nonzero()[:, 0]
        pos = self.positions[t].long()
        return t, pos, self.tables[self.seqs[t].long(), pos // self.page].long(), pos % self.page

    def verify(self, K0, V0):
        t, pos, page, row = self.live()
        u = unit(self.dtype)
        tiny = 2.0 ** -25 if self.dtype == F16 else 0.0

        def near(got, x, w, what):
            y, off = append_reference(x, w, EPS, self.cos, self.sin, pos)
            # the sum off an exact y, then half a step of what is rounded
            assert bool(((got.double() - y).abs() <= off + u * (y.abs() + off) + tiny).all()), what

        rest = torch.ones(self.T, dtype=torch.bool, device=DEV)
        rest[t] = False
        for out in (self.q_out, self.k_out, self.v_out):
            assert bool((out[rest] == 7.0).all())            # padding writes nothing
        near(self.q_out[t], self.q[t], self.wq, "q_out")
        if self.fmt == "mxfp4":
            k, _ = append_reference(self.k[t], self.wk, EPS, self.cos, self.sin, pos)
            for pool, old, x, out in ((self.K, K0, k, self.k_out), (self.V, V0, self.v[t].double(), self.v_out)):
                code, scale = quantise(x, self.dtype)
                c, s = unpack(old.clone(), self.page, self.D)
                c[page, :, row], s[page, :, row] = code, scale
                gc, gs = unpack(pool, self.page, self.D)
                assert torch.equal(gs, s) and torch.equal(gc, c)
                assert torch.equal(out[t].double(), values(code, scale))
        else:
            K, V = K0.clone(), V0.clone()
            near(self.k_out[t], self.k[t], self.wk, "k_out")
            K[page, :, row], V[page, :, row] = self.k_out[t], self.v[t]
            assert torch.equal(self.K, K) and torch.equal(self.V, V) and torch.equal(self.v_out[t], self.v[t])

    def go(self, **kw):
        K0, V0 = self.K.clone(), self.V.clone()
        assert self.run(**kw) is self.q_out
        self.verify(K0, V0)


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True), (False, False)])
def test_forms(norm, rope, D, dtype, fmt):
    Call([1, 17, 0, 40, 5], [0, 30, 9, 15, 255], 8, 2, D, dtype, 16, fmt, norm, rope, seed=D + norm, padding=3).go()


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (12, 12), (20, 4), (7, 7), (40, 8)])
def test_heads_and_pages(heads, page, fmt):
    Call([33, 1, 64], [0, 100, 250], *heads, 64 if heads[0] % 2 else 128, BF16, page, fmt, seed=page).go()


@pytest.mark.parametrize("T", [1, 2, 3, 255, 256, 257, 3000])
def test_steps(T):
    """One token per sequence, seqs left out: token t is sequence t's."""
    c = Call([1] * T, [(7 * i) % 300 for i in range(T)], 4, 2, 64, F16, 32, "16", seed=T)
    order = torch.argsort(c.seqs)
    c.seqs, c.positions = c.seqs[order], c.positions[order]
    assert torch.equal(c.seqs, torch.arange(T, dtype=torch.int32, device=DEV))
    c.go(seqs=None)


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_long_prompts(fmt):
    Call([4099, 2048, 1], [0, 777, 5000], 16, 4, 128, BF16, 64, fmt, seed=1).go()


def test_bits_of_the_contiguous_append():
    """fp16 without norms: the rows that cdna3_rope_append_kv_f16 writes."""
    c = Call([50], [0], 8, 2, 64, F16, 16, "16", norm=False, seed=2)
    order = torch.argsort(c.positions)
    c.q, c.k, c.v, c.positions = c.q[order].contiguous(), c.k[order].contiguous(), c.v[order].contiguous(), c.positions[order]
    c.run()
    qh = torch.empty(8, 50, 64, dtype=F16, device=DEV)
    Kc, Vc = torch.empty(2, 50, 64, dtype=F16, device=DEV), torch.empty(2, 50, 64, dtype=F16, device=DEV)
    cdna4.rope_append_kv_f16(c.q, c.k, c.v, qh, Kc, Vc, c.cos[:50].contiguous(), c.sin[:50].contiguous(), 50, 8, 2, 64, 0, 50)
    assert torch.equal(c.q_out, qh.transpose(0, 1)) and torch.equal(c.k_out, Kc.transpose(0, 1)) and torch.equal(c.v_out, Vc.transpose(0, 1))


def test_in_place_and_without_queries():
    for fmt in ("16", "mxfp4"):
        a = Call([20, 9], [3, 40], 8, 2, 128, F16, 16, fmt, seed=3)
        K, V = a.K.clone(), a.V.clone()
        a.run()
        q, k, v = a.q.clone(), a.k.clone(), a.v.clone()       # packed copies, then the outputs in their place
        cdna4.rope_append_paged(q, k, v, K, V, a.tables, a.positions, a.cache, q, seqs=a.seqs, cos=a.cos, sin=a.sin, q_norm=a.wq, k_norm=a.wk,
                                eps=EPS, k_out=k, v_out=v)
        assert torch.equal(q, a.q_out) and torch.equal(k, a.k_out) and torch.equal(v, a.v_out) and torch.equal(K, a.K) and torch.equal(V, a.V)
        K.fill_(0), V.fill_(0)
        t, _, page, row = a.live()
        assert cdna4.rope_append_paged(None, a.k, a.v, K, V, a.tables, a.positions, a.cache, seqs=a.seqs, cos=a.cos, sin=a.sin, k_norm=a.wk, eps=EPS) is None
        pick = lambda p: p[page, :, row] if fmt == "16" else unpack(p, 16, 128)[0][page, :, row]
        assert torch.equal(pick(K), pick(a.K)) and torch.equal(pick(V), pick(a.V))


def test_padding_of_every_kind():
    """Sequences and positions outside their ranges write nothing; a missing page leaves the pools alone and gives the outputs."""
    c = Call([6], [0], 4, 2, 64, F16, 16, "16", seed=4)
    order = torch.argsort(c.positions)
    c.q, c.k, c.v, c.positions, c.seqs = c.q[order], c.k[order], c.v[order], c.positions[order], c.seqs[order]
    c.seqs.copy_(torch.tensor([-1, 1, 2 ** 31 - 1, 0, 0, 0], dtype=torch.int32))
    c.positions.copy_(torch.tensor([0, 1, 2, -1, 2 ** 31 - 1, 16], dtype=torch.int32))   # the last lies in the table's empty entry
    c.cos, c.sin = cdna4.rope_table_f32(0, 40, 64, 10000.0, device=DEV)
    K0, V0 = c.K.clone(), c.V.clone()
    c.run()
    assert torch.equal(c.K, K0) and torch.equal(c.V, V0)
    assert bool((c.q_out[:5] == 7).all()) and bool((c.k_out[:5] == 7).all()) and bool((c.v_out[:5] == 7).all())
    y, off = append_reference(c.q[5:], c.wq, EPS, c.cos, c.sin, torch.tensor([16], device=DEV))
    assert bool(((c.q_out[5:].double() - y).abs() <= off + 2.0 ** -11 * (y.abs() + off) + 2.0 ** -25).all())
    for bad in (10 ** 6, -3):                                # pages outside the pool
        c.tables[0, 1] = bad
        c.run()
        assert torch.equal(c.K, K0) and torch.equal(c.V, V0)
    # positions past the angles are padding too
    c.q_out.fill_(7.0)
    c.seqs.zero_()
    c.positions.copy_(torch.tensor([40, 39, 41, 50, 60, 70], dtype=torch.int32))
    c.run(cos=c.cos[:39].contiguous(), sin=c.sin[:39].contiguous())
    assert bool((c.q_out == 7).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_4_bit_blocks_of_every_size(dtype, D):
    """Rows of zeros, of the type's smallest and largest values, and with values that are not finite in one block."""
    c = Call([24], [0], 2, 2, D, dtype, 16, "mxfp4", norm=False, rope=False, seed=5)
    big = torch.finfo(dtype).max
    small = 2.0 ** -24 if dtype == F16 else 2.0 ** -133
    for x in (c.k, c.v):
        for t, s in enumerate((0.0, small, 8 * small, big, big / 4, 7.0, 6.99, 2.0 ** -14, 1e-3)):
            x[t] = (x[t].double().clamp(-1, 1) * s).to(dtype)
            x[t, :, 0] = s
            x[t, :, 33] = -s
        for t, bad in ((10, float("inf")), (11, -float("inf")), (12, float("nan"))):
            x[t, 0, 40] = bad
    K0, V0 = c.K.clone(), c.V.clone()
    c.run()
    t, pos, page, row = c.live()
    for pool, old, x, out in ((c.K, K0, c.k, c.k_out), (c.V, V0, c.v, c.v_out)):
        code, scale = quantise(x[t], dtype)
        gc, gs = unpack(pool, 16, D)
        assert torch.equal(gs[page, :, row], scale) and torch.equal(gc[page, :, row], code)
        want = values(code, scale)
        got = out[t].double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert int(want.isnan().sum()) == 3 * 32


def test_captured_call_replays_on_other_positions():
    c = Call([1] * 8, list(range(0, 240, 30)), 4, 2, 64, BF16, 16, "mxfp4", seed=6, later=3)
    c.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    for step in range(1, 4):
        c.positions += 1
        c.k.mul_(-0.5)
        K0, V0 = c.K.clone(), c.V.clone()
        c.q_out.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        c.verify(K0, V0)


def test_another_stream():
    c = Call([100, 30], [0, 7], 8, 2, 128, F16, 32, "16", seed=7)
    K0, V0 = c.K.clone(), c.V.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    c.run(stream=s)
    torch.cuda.synchronize()
    c.verify(K0, V0)


def test_python_refuses():
    c = Call([4], [0], 4, 2, 64, F16, 16, "16", seed=8)
    bad = [dict(cos=None), dict(sin=None), dict(q_norm=c.wq[:32]), dict(k_norm=c.wq.to(BF16)), dict(k_out=c.k_out[:3]), dict(v_out=c.v_out.to(BF16)),
           dict(seqs=c.seqs[:2]), dict(cos=c.cos.double(), sin=c.sin.double()), dict(cos=c.cos[:, :32].contiguous(), sin=c.sin[:, :32].contiguous())]
    for kw in bad:
        with pytest.raises(ValueError):
            c.run(**kw)
    with pytest.raises(ValueError):
        cdna4.rope_append_paged(c.q, c.k, c.v, c.K[:1], c.V, c.tables, c.positions, c.cache, c.q_out, seqs=c.seqs)
    with pytest.raises(ValueError):
        cdna4.rope_append_paged(None, c.k, c.v, c.K, c.V, c.tables, c.positions, c.cache, c.q_out, seqs=c.seqs)
    with pytest.raises(ValueError):                          # four tokens, one table
        c.run(seqs=None)


@pytest.mark.parametrize("name", ["q", "k", "v", "q_out", "k_out", "v_out"])
def test_tokens_over_each_other_are_refused(name):
    """One token's row repeated by expand() has a token stride of 0, which the C call would take for packed tokens."""
    c = Call([5], [0], 4, 2, 64, F16, 16, "16", seed=10)
    K0, V0, t = c.K.clone(), c.V.clone(), getattr(c, name)
    setattr(c, name, t[:1].contiguous().expand(t.shape))
    with pytest.raises(ValueError):
        c.run()
    assert torch.equal(c.K, K0) and torch.equal(c.V, V0)
    # one token may have any stride
    one = dict(seqs=c.seqs[:1], k_out=c.k_out[:1], v_out=c.v_out[:1])
    cdna4.rope_append_paged(c.q[:1], c.k[:1], c.v[:1], c.K, c.V, c.tables, c.positions[:1], c.cache, c.q_out[:1], cos=c.cos, sin=c.sin, **one)


def test_pools_past_32_bit_offsets():
    HK, D, page = 8, 128, 256
    pages = 2 ** 32 // (HK * page * 256) + 8
    c = Call([40], [250], 8, HK, D, F16, page, "16", seed=9)
    for name in ("K", "V"):
        setattr(c, name, torch.zeros(pages, HK, page, D, dtype=F16, device=DEV))
    c.tables = torch.where(c.tables >= 0, c.tables + pages - c.cache.pages, c.tables)
    c.cache.pages = pages
    c.run()
    t, pos, pg, row = c.live()
    assert torch.equal(c.K[pg, :, row], c.k_out[t]) and torch.equal(c.V[pg, :, row], c.v[t])
    assert int((c.V != 0).any(-1).sum()) == 40 * HK
