"""The paged cache's calls together, as a program would use them: prompts appended with norms and rotation, their own attention in a packed
call over what the cache now holds, then beam search: a step's tokens appended, attention over the pages, the vocabulary product,
selection, reordering, pages given out as the sequences grow."""
import math

import pytest
import torch

import cdna4
from paged_util import decode_reference
from serving_util import DEV, check, cu_of, packed_reference

pytestmark = pytest.mark.gpu
F16 = torch.float16
G, BEAMS, HQ, HK, D, PAGE, V = 3, 4, 8, 2, 64, 16, 4096
ROWS, WIDTH, POOL = G * BEAMS, 8, 200


class Model:
    """A one-layer stand-in for a decoder: token embeddings projected to q, k, v, and attention's output to logits."""

    def __init__(self, fmt, seed=0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        r = lambda *s: torch.randn(*s, device=DEV, generator=g)
        self.qkv = r(V, HQ + 2 * HK, D).to(F16)
        self.out = (4 * r(V, HQ * D) / math.sqrt(HQ * D)).to(F16)
        self.norms = [(1 + 0.1 * r(D)).to(F16) for _ in range(2)]
        self.cos, self.sin = cdna4.rope_table_f32(0, WIDTH * PAGE, D, 10000.0, device=DEV)
        self.cache = cdna4.PagedCache(D, HK, PAGE, POOL, cdna4.KV_MXFP4 if fmt == "mxfp4" else cdna4.KV_16BIT, WIDTH)
        shape = cdna4.paged_pool_shape(self.cache)
        if fmt == "mxfp4":
            self.K, self.V = (torch.full(shape, 255, dtype=torch.uint8, device=DEV) for _ in range(2))
        else:
            self.K, self.V = (torch.full(shape, float("nan"), dtype=F16, device=DEV) for _ in range(2))

    def append(self, ids, tables, positions, seqs=None, q_out=None, k_out=None, v_out=None):
        x = self.qkv[ids]
        return cdna4.rope_append_paged(x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:], self.K, self.V, tables, positions, self.cache, q_out, seqs=seqs,
                                       cos=self.cos, sin=self.sin, q_norm=self.norms[0], k_norm=self.norms[1], k_out=k_out, v_out=v_out)


i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_prompts_then_beams(fmt):
    m = Model(fmt)
    free = list(range(POOL))
    prompts = [torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(n)).to(DEV) for n in (1, 33, 16)]
    lens = [len(p) for p in prompts]
    tables = torch.full((ROWS, WIDTH), -1, dtype=torch.int32)
    for g, n in enumerate(lens):
        for j in range((n + PAGE - 1) // PAGE):
            tables[g * BEAMS, j] = free.pop()
    tables = tables.to(DEV)
    # prompts: into the pages of each group's first beam, and attended over in one packed call
    T, cu = sum(lens), cu_of(lens)
    k, v = (torch.empty(T, HK, D, dtype=F16, device=DEV) for _ in range(2))
    q = m.append(torch.cat(prompts), tables, torch.cat([torch.arange(n) for n in lens]).int().to(DEV),
                 seqs=i32([g * BEAMS for g, n in enumerate(lens) for _ in range(n)]), k_out=k, v_out=v)
    O = torch.empty(T, HQ, D, dtype=F16, device=DEV)
    cdna4.prefill_packed(q, k, v, O, i32(cu), cdna4.PackedPrefillCfg(D, HQ, HK, G, T, max(lens), 0, 0))
    ref, bound, _ = packed_reference(q, k, v, cu, D, HQ // HK, F16)
    check(O, ref, bound, "prompts")
    # the last tokens once more by the paged call: the same rows
    one = cdna4.PagedDecodeCfg(HQ, G, 1)
    o = torch.empty(G, 1, HQ, D, dtype=F16, device=DEV)
    ends = [c - 1 for c in cu[1:]]
    cdna4.decode_paged(q[ends].unsqueeze(1).contiguous(), m.K, m.V, tables[::BEAMS].contiguous(), i32(lens), o, m.cache, one)
    check(o[:, 0], O[ends].double(), 2 * bound[ends], "prompts by pages")
    held = [(k[cu[r // BEAMS]:cu[r // BEAMS + 1]], v[cu[r // BEAMS]:cu[r // BEAMS + 1]]) for r in range(ROWS)]

    logits = cdna4.gemm_f16_nt(O[ends].reshape(G, HQ * D), m.out, out_dtype=torch.float32).repeat_interleave(BEAMS, 0)
    cum = torch.tensor([0.0] + [-math.inf] * (BEAMS - 1), device=DEV).repeat(G)
    length = i32([n for n in lens for _ in range(BEAMS)])
    cfg = cdna4.PagedDecodeCfg(HQ, ROWS, 1)
    ws = torch.empty(cdna4.decode_paged_workspace_size(m.cache, cfg), dtype=torch.uint8, device=DEV)
    said = [[] for _ in range(ROWS)]
    for step in range(20):
        score, parent, token = cdna4.beam_select(logits, cum, BEAMS)
        # 64-bit: every row's continuations, all of the group's sorted
        x = logits.double() - torch.logsumexp(logits.double(), 1, keepdim=True) + cum.double()[:, None]
        best = x.view(G, -1).topk(BEAMS).values
        assert float((score.double() - best).abs().max()) < 1e-4
        at = x.view(G, -1).gather(1, ((parent % BEAMS).long() * V + token.long()))
        assert float((at - best).abs().max()) < 1e-9          # the places named are those of the best ones
        cum, par, tok = score.reshape(-1).contiguous(), parent.reshape(-1).contiguous(), token.reshape(-1)
        fresh = [free.pop(0) for _ in range(ROWS)]
        to, lo = torch.empty_like(tables), torch.empty_like(length)
        cdna4.paged_reorder(par, tables, length, i32(fresh), to, lo, m.K, m.V, m.cache)
        tables, length = to, lo
        held = [held[p] for p in par.tolist()]
        said = [said[p] + [t] for p, t in zip(par.tolist(), tok.tolist())]
        n = length.tolist()
        for r in range(ROWS):                                # a page for the rows whose last one is full
            if n[r] % PAGE == 0:
                tables[r, n[r] // PAGE] = fresh[r]
        k, v = (torch.empty(ROWS, HK, D, dtype=F16, device=DEV) for _ in range(2))
        q = m.append(tok.long(), tables, length.clone(), k_out=k, v_out=v)
        length += 1
        held = [(torch.cat([a, k[r:r + 1]]), torch.cat([b, v[r:r + 1]])) for r, (a, b) in enumerate(held)]
        o = torch.empty(ROWS, 1, HQ, D, dtype=F16, device=DEV)
        cdna4.decode_paged(q, m.K, m.V, tables, length, o, m.cache, cfg, workspace=ws)
        ref, bound = decode_reference(q.unsqueeze(1), [a.transpose(0, 1) for a, _ in held], [b.transpose(0, 1) for _, b in held], F16)
        check(o, ref, bound, f"step {step}")
        used = {int(p) for r in range(ROWS) for p in tables[r, :(int(length[r]) + PAGE - 1) // PAGE]}
        free = [p for p in range(POOL) if p not in used]
        logits = cdna4.gemm_f16_nt(o.view(ROWS, HQ * D), m.out, out_dtype=torch.float32)
    for g in range(G):                                       # the beams of a group differ
        assert len({tuple(s) for s in said[g * BEAMS:(g + 1) * BEAMS]}) == BEAMS


@pytest.mark.parametrize("fmt", ["16", "mxfp4"])
def test_step_as_a_graph(fmt):
    """A captured step (append, attention, vocabulary product, selection, reordering) replayed while the program's own eager calls go on
    between the replays; every replay equals the eager step bit for bit."""
    m = Model(fmt, 1)
    tables = torch.arange(ROWS * 4, dtype=torch.int32, device=DEV).view(ROWS, 4)
    tables = torch.cat([tables, torch.full((ROWS, WIDTH - 4), -1, dtype=torch.int32, device=DEV)], 1)
    fresh = torch.arange(ROWS * 4, ROWS * 5, dtype=torch.int32, device=DEV)
    for t in range(40):                                      # what the cache holds at first
        m.append(torch.randint(0, V, (ROWS,), device=DEV), tables, i32([t] * ROWS))
    cfg = cdna4.PagedDecodeCfg(HQ, ROWS, 1)
    size, bsize = cdna4.decode_paged_workspace_size(m.cache, cfg), cdna4.beam_select_workspace_size(ROWS, V, BEAMS, BEAMS)

    class Step:
        def __init__(self, token, length, cum, K, V_):
            self.token, self.length, self.cum, self.K, self.V = token, length, cum, K, V_
            self.q, self.o = torch.zeros(ROWS, HQ, D, dtype=F16, device=DEV), torch.zeros(ROWS, 1, HQ, D, dtype=F16, device=DEV)
            self.logits = torch.zeros(ROWS, V, device=DEV)
            self.out = tuple(torch.zeros(G, BEAMS, dtype=d, device=DEV) for d in (torch.float32, torch.int32, torch.int32))
            self.to, self.lo = torch.zeros_like(tables), torch.zeros_like(length)
            self.ws, self.bws = (torch.empty(n, dtype=torch.uint8, device=DEV) for n in (size, bsize))

        def run(self):
            x = m.qkv[self.token]
            cdna4.rope_append_paged(x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:], self.K, self.V, tables, self.length, m.cache, self.q, cos=m.cos,
                                    sin=m.sin, q_norm=m.norms[0], k_norm=m.norms[1])
            n = self.length + 1
            cdna4.decode_paged(self.q, self.K, self.V, tables, n, self.o, m.cache, cfg, workspace=self.ws)
            cdna4.gemm_f16_nt(self.o.view(ROWS, HQ * D), m.out, out=self.logits)
            cdna4.beam_select(self.logits, self.cum, BEAMS, out=self.out, workspace=self.bws)
            cdna4.paged_reorder(self.out[1].view(-1), tables, n, fresh, self.to, self.lo, self.K, self.V, m.cache)

        def results(self):
            bits = lambda t: t.view(torch.uint8 if t.dtype == torch.uint8 else torch.int16)
            return self.q, self.o, self.logits, *self.out, self.to, self.lo, bits(self.K), bits(self.V)

    g = Step(torch.randint(0, V, (ROWS,), device=DEV), i32([40] * ROWS), torch.zeros(ROWS, device=DEV), m.K.clone(), m.V.clone())
    g.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.run()
    for i in range(4):
        g.token.copy_(torch.randint(0, V, (ROWS,), device=DEV))
        g.length.copy_(torch.randint(1, 62, (ROWS,), device=DEV).int())
        g.cum.copy_(-5 * torch.rand(ROWS, device=DEV))
        g.K.copy_(m.K), g.V.copy_(m.V)
        e = Step(g.token.clone(), g.length.clone(), g.cum.clone(), m.K.clone(), m.V.clone())
        graph.replay()
        e.run()
        torch.cuda.synchronize()
        for a, b in zip(g.results(), e.results()):
            assert torch.equal(a.nan_to_num() if a.is_floating_point() else a, b.nan_to_num() if b.is_floating_point() else b), i


def test_tables_wider_than_max_pages():
    """Refused without a table_stride, whose rows the calls would read at the wrong places; with one, the packed tables' bits."""
    m = Model("16", 2)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    order = torch.randperm(POOL, device=DEV, generator=g).int()
    tables, wide = order[:ROWS * 4].view(ROWS, 4).contiguous(), torch.full((ROWS, WIDTH), -1, dtype=torch.int32, device=DEV)
    wide[:, :4] = tables
    n, fresh = torch.randint(1, 64, (ROWS,), device=DEV, generator=g).int(), order[ROWS * 4:ROWS * 5].contiguous()
    parents = torch.randint(0, ROWS, (ROWS,), device=DEV, generator=g).int()
    ids, cfg = torch.randint(0, V, (ROWS,), device=DEV, generator=g), cdna4.PagedDecodeCfg(HQ, ROWS, 1)
    for t in range(64):                                      # rows for every length
        m.append(ids, wide, i32([t] * ROWS))
    K0, V0 = m.K, m.V

    def step(tables, stride, outs):
        m.cache.max_pages, m.cache.table_stride, m.K, m.V = 4, stride, K0.clone(), V0.clone()
        lens_out, o = torch.zeros_like(n), torch.zeros(ROWS, 1, HQ, D, dtype=F16, device=DEV)
        q = m.append(ids, tables, n - 1)
        cdna4.decode_paged(q, m.K, m.V, tables, n, o, m.cache, cfg)
        cdna4.paged_reorder(parents, tables, n, fresh, outs, lens_out, m.K, m.V, m.cache)
        return q, o, outs[:, :4], lens_out, m.K.nan_to_num(), m.V.nan_to_num()

    a, b = step(tables, 0, torch.zeros_like(tables)), step(wide, WIDTH, torch.zeros_like(wide))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    q, o = a[0], a[1]
    m.cache.table_stride = 0
    for call in (lambda: m.append(ids, wide, n - 1), lambda: cdna4.decode_paged(q, m.K, m.V, wide, n, o, m.cache, cfg),
                 lambda: cdna4.paged_reorder(parents, wide, n, fresh, tables, n.clone(), m.K, m.V, m.cache),
                 lambda: cdna4.paged_reorder(parents, tables, n, fresh, wide, n.clone(), m.K, m.V, m.cache)):
        with pytest.raises(ValueError):
            call()
