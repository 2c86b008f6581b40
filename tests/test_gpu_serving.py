"""The batched serving calls together, as a program would use them: prompts of different lengths behind one system
prompt in a packed call, their keys into caches, then steps of one token for the whole batch: shared-prefix attention,
the vocabulary product, penalties and masks, probabilities, the next token."""
import math

import pytest
import torch

import cdna4
from serving_util import DEV, check, cu_of, packed_reference, shared_reference

pytestmark = pytest.mark.gpu
F16 = torch.float16
B, HQ, HK, D, P, CAP, V = 5, 8, 2, 64, 150, 96, 4096
G = HQ // HK


class Batch:
    """A one-layer stand-in for a decoder: token embeddings projected to q, k, v, and attention's output to logits."""

    def __init__(self, seed=0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        r = lambda *s: torch.randn(*s, device=DEV, generator=g)
        self.qkv = r(V, HQ + 2 * HK, D).to(F16)                       # per token, as a projection would give them
        self.out = (r(V, HQ * D) / math.sqrt(HQ * D)).to(F16)
        self.system = torch.randint(0, V, (P,), device=DEV, generator=g)
        self.prompts = [torch.randint(0, V, (n,), device=DEV, generator=g) for n in (1, 33, 64, 7, 50)]
        x = self.qkv[self.system]
        self.Kp = x[:, HQ:HQ + HK].transpose(0, 1).contiguous()
        self.Vp = x[:, HQ + HK:].transpose(0, 1).contiguous()

    def prefill(self):
        lens = [len(p) for p in self.prompts]
        x = self.qkv[torch.cat(self.prompts)]
        Q, K, Vv = x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:]
        cu = cu_of(lens)
        O = torch.empty(len(x), HQ, D, dtype=F16, device=DEV)
        cfg = cdna4.PackedPrefillCfg(D, HQ, HK, B, len(x), max(lens), P, 0)
        cdna4.prefill_packed(Q, K, Vv, O, torch.tensor(cu, dtype=torch.int32, device=DEV), cfg, self.Kp, self.Vp)
        self.Kc = torch.full((B, HK, CAP, D), float("nan"), dtype=F16, device=DEV)
        self.Vc = torch.full((B, HK, CAP, D), float("nan"), dtype=F16, device=DEV)
        for b in range(B):
            self.Kc[b, :, :lens[b]] = K[cu[b]:cu[b + 1]].transpose(0, 1)
            self.Vc[b, :, :lens[b]] = Vv[cu[b]:cu[b + 1]].transpose(0, 1)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        return Q, K, Vv, O, cu


def test_prompts_then_steps():
    m = Batch()
    Q, K, Vv, O, cu = m.prefill()
    ref, bound, _ = packed_reference(Q, K, Vv, cu, D, G, F16, m.Kp, m.Vp, P)
    check(O, ref, bound, "prompts")

    cfg = cdna4.SharedDecodeCfg(D, HQ, HK, B, P, 0, CAP, 0)
    ws = torch.empty(cdna4.decode_shared_workspace_size(cfg), dtype=torch.uint8, device=DEV)
    history = torch.full((B, CAP), -1, dtype=torch.int32, device=DEV)
    plen = m.lens.clone()
    for b, p in enumerate(m.prompts):
        history[b, :len(p)] = p.int()
    pen = dict(repetition=torch.full((B,), 1.3, device=DEV), frequency=torch.full((B,), 0.2, device=DEV),
               presence=torch.full((B,), 0.1, device=DEV))
    # a grammar that allows even tokens only in the first sequence
    mask = torch.full((B, V // 32), -1, dtype=torch.int32, device=DEV)
    mask[0] = 0x55555555
    bias_ids = torch.full((B, 2), -1, dtype=torch.int32, device=DEV)
    bias_values = torch.zeros(B, 2, device=DEV)
    bias_ids[3, 0], bias_values[3, 0] = 77, 1e4          # the fourth is made to say 77
    token = torch.stack([p[-1] for p in m.prompts])
    seqs = [p.tolist() for p in m.prompts]
    for step in range(6):
        # the last token's own k and v are in the cache from the second step on
        if step:
            x = m.qkv[token]
            at = m.lens.long()
            rows = torch.arange(B, device=DEV)
            m.Kc[rows, :, at] = x[:, HQ:HQ + HK]
            m.Vc[rows, :, at] = x[:, HQ + HK:]
            m.lens += 1
        q = m.qkv[token][:, :HQ].contiguous()
        o = torch.empty(B, HQ, D, dtype=F16, device=DEV)
        cdna4.decode_shared(q, m.Kp, m.Vp, m.Kc, m.Vc, m.lens, o, cfg, workspace=ws)
        lens = m.lens.tolist()
        ref, bound = shared_reference(q, m.Kp, m.Vp, m.Kc, m.Vc, lens, G, F16, P)
        check(o, ref, bound, f"step {step}")
        # the same rows as a packed call over the whole sequences gives them
        ids = [torch.tensor(s, device=DEV) for s in seqs]
        x = m.qkv[torch.cat(ids)]
        cu = cu_of(lens)
        Op = torch.empty(len(x), HQ, D, dtype=F16, device=DEV)
        cdna4.prefill_packed(x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:], Op, torch.tensor(cu, dtype=torch.int32, device=DEV),
                             cdna4.PackedPrefillCfg(D, HQ, HK, B, len(x), max(lens), P, 0), m.Kp, m.Vp)
        check(o, Op[[c - 1 for c in cu[1:]]].double(), 2 * bound, f"step {step} against the packed call")

        logits = cdna4.gemm_f16_nt(o.view(B, HQ * D), m.out, out_dtype=F16)
        x = cdna4.process_logits(logits, history=history, history_len=m.lens, prompt_len=plen, mask=mask, bias_ids=bias_ids,
                                 bias_values=bias_values, **pen)
        probs = cdna4.softmax_rows_f32(x)
        # 64-bit from the same logits
        y = logits.double()
        for b in range(B):
            h = history[b, :lens[b]].long()
            seen = torch.unique(h)
            v = y[b, seen]
            y[b, seen] = torch.where(v > 0, v / pen["repetition"][b].double(), v * pen["repetition"][b].double())
            made, n = torch.unique(h[int(plen[b]):], return_counts=True)
            y[b, made] -= n.double() * pen["frequency"][b].double() + pen["presence"][b].double()
        y[3, 77] += 1e4
        y[0, 1::2] = -math.inf
        want = torch.softmax(y, 1)
        assert bool((probs[0, 1::2] == 0).all()) and float(probs[3, 77]) == 1.0
        # exp's argument is off by a few roundings of logits below 2^5 (2^14 in the biased row, whose softmax is exact)
        assert float((probs.double() - want).abs().max()) <= 2.0 ** -24 * 2 ** 5 * 16
        token = probs.argmax(1)
        top = y.gather(1, token[:, None])[:, 0]
        assert bool((top >= y.amax(1) - 1e-4).all())
        for b in range(B):
            seqs[b].append(int(token[b]))
        history[torch.arange(B, device=DEV), m.lens.long()] = token.int()
    assert all(t % 2 == 0 for t in seqs[0][1:]) and seqs[3][-1] == 77


def test_step_as_a_graph():
    """A captured step (attention, vocabulary product, logits) replayed while the program's own eager calls go on
    between the replays; every replay equals the eager step bit for bit."""
    m = Batch(1)
    m.prefill()
    cfg = cdna4.SharedDecodeCfg(D, HQ, HK, B, P, 0, CAP, 0)
    ws = torch.empty(cdna4.decode_shared_workspace_size(cfg), dtype=torch.uint8, device=DEV)
    token = torch.stack([p[-1] for p in m.prompts])
    q = m.qkv[token][:, :HQ].contiguous()
    o = torch.empty(B, HQ, D, dtype=F16, device=DEV)
    logits = torch.empty(B, V, dtype=F16, device=DEV)
    x = torch.empty(B, V, device=DEV)
    history = torch.randint(0, V, (B, CAP), device=DEV).int()
    rep = torch.full((B,), 1.2, device=DEV)

    def step(q, o, logits, x, ws):
        cdna4.decode_shared(q, m.Kp, m.Vp, m.Kc, m.Vc, m.lens, o, cfg, workspace=ws)
        cdna4.gemm_f16_nt(o.view(B, HQ * D), m.out, out=logits)
        return cdna4.process_logits(logits, x, history=history, history_len=m.lens, repetition=rep)

    step(q, o, logits, x, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, o, logits, x, ws)
    for i in range(4):
        m.Kc[:, :, CAP - 8:] = 0.5
        m.Vc[:, :, CAP - 8:] = -0.25
        m.lens.copy_(torch.tensor([1 + i, 20, 64 - i, 7, 50], dtype=torch.int32))
        token = torch.randint(0, V, (B,), device=DEV)
        q.copy_(m.qkv[token][:, :HQ])
        x.fill_(7.0)
        graph.replay()
        m2 = step(q.clone(), torch.empty_like(o), torch.empty_like(logits), torch.empty_like(x), torch.empty_like(ws))
        torch.cuda.synchronize()
        # as bits: the first sequence, longer here than its prompt, reads rows of its cache that still hold NaN
        assert torch.equal(x.view(torch.int32), m2.view(torch.int32)), i
