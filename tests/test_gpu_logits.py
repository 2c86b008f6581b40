"""cdna4.process_logits against a 64-bit reference: odd vocabularies, empty and full histories, repeated ids and
padding, biases, masks that leave nothing, logits of every value."""
import math

import pytest
import torch

import cdna4
from serving_util import DEV

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def reference(logits, history=None, history_len=None, prompt_len=None, repetition=None, frequency=None, presence=None,
              bias_ids=None, bias_values=None, mask=None):
    """(x, bound): float64 values and what fp32 arithmetic may be off by. Four operations after the exact
    widening, each rounded once (2^-24 relative) on a value no larger than the sum of the parts' sizes."""
    x = logits.double().cpu().clone()
    M, V = x.shape
    size = x.abs()
    for m in range(M):
        if history is not None:
            n = history.shape[1] if history_len is None else min(max(int(history_len[m]), 0), history.shape[1])
            p = 0 if prompt_len is None else min(max(int(prompt_len[m]), 0), n)
            r = 1.0 if repetition is None else float(repetition[m])
            f = 0.0 if frequency is None else float(frequency[m])
            q = 0.0 if presence is None else float(presence[m])
            ids = history[m, :n].cpu().tolist()
            for t in {t for t in ids if 0 <= t < V}:
                c = sum(1 for u in ids[p:] if u == t)
                v = float(x[m, t])
                v = v / r if v > 0 else v * r
                size[m, t] = abs(v) + c * abs(f) + (abs(q) if c else 0)
                x[m, t] = v - c * f - (q if c else 0)
        if bias_ids is not None:
            last = {}
            for t, b in zip(bias_ids[m].tolist(), bias_values[m].tolist()):
                if 0 <= t < V:
                    last[t] = b
            for t, b in last.items():
                x[m, t] += b
                size[m, t] += abs(b)
    bound = size * 4 * 2.0 ** -24
    if mask is not None:
        words = mask.cpu().long()
        j = torch.arange(V)
        x[((words[:, j // 32] >> (j % 32)) & 1) == 0] = -math.inf
    return x, bound


def check(got, x, bound):
    got = got.double().cpu()
    fin = torch.isfinite(x)
    assert torch.equal(torch.isnan(got), torch.isnan(x))
    odd = ~fin & ~torch.isnan(x)
    assert torch.equal(got[odd], x[odd])
    d = (got - x)[fin].abs()
    assert bool((d <= bound[fin]).all()), float((d - bound[fin]).max())


def inputs(M, V, H, dtype, seed=0, hot=None):
    g = torch.Generator().manual_seed(seed)
    u = lambda *s: torch.rand(*s, generator=g)
    hot = hot or V
    kw = dict(history=torch.randint(-1, min(hot, V) + 1, (M, H), generator=g).int(), history_len=(u(M) * (H + 1)).int().clamp(max=H),
              repetition=1 + u(M), frequency=u(M) - 0.3, presence=u(M) - 0.3)
    kw["prompt_len"] = (u(M) * (kw["history_len"] + 1)).int()
    logits = (torch.randn(M, V, generator=g) * 5).to(dtype)
    return logits.to(DEV), {k: v.to(DEV) for k, v in kw.items()}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,V,H", [(1, 1, 1), (3, 7, 5), (2, 8, 40), (5, 33, 0), (4, 1000, 300), (3, 8191, 1000), (2, 8193, 77),
                                   (2, 32000, 513), (65, 1025, 20), (1, 100003, 4000)])
def test_penalties(M, V, H, dtype):
    logits, kw = inputs(M, V, H, dtype, seed=V + H, hot=max(4, H // 2))
    check(cdna4.process_logits(logits, **kw), *reference(logits, **kw))


def test_many_rows_large_chunks():
    logits, kw = inputs(300, 40001, 50, BF16, seed=5, hot=30)
    out = cdna4.process_logits(logits, **kw)
    pick = [0, 1, 137, 298, 299]
    sub = {k: v[pick] for k, v in kw.items()}
    check(out[pick], *reference(logits[pick], **sub))


@pytest.mark.parametrize("part", ["repetition", "frequency", "presence", "none"])
def test_single_penalties_and_defaults(part):
    logits, kw = inputs(4, 500, 60, F16, seed=1, hot=50)
    keep = {"history": kw["history"]} if part == "none" else {"history": kw["history"], part: kw[part]}
    check(cdna4.process_logits(logits, **keep), *reference(logits, **keep))
    check(cdna4.process_logits(logits), *reference(logits))


@pytest.mark.parametrize("lens", [(0, 0), (60, 0), (60, 60), (-5, 3), (1000, -4), (1, 1), (30, 99)])
def test_lengths_are_cut(lens):
    logits, kw = inputs(2, 400, 60, F32, seed=2, hot=20)
    kw["history_len"].fill_(lens[0])
    kw["prompt_len"].fill_(lens[1])
    check(cdna4.process_logits(logits, **kw), *reference(logits, **kw))


def test_one_token_all_along():
    """Every entry the same id: one counter takes them all."""
    logits, kw = inputs(3, 9000, 5000, F32, seed=3)
    kw["history"].fill_(8200)
    kw["history_len"].fill_(5000)
    kw["prompt_len"].copy_(torch.tensor([0, 2500, 5000]))
    check(cdna4.process_logits(logits, **kw), *reference(logits, **kw))


def test_biases():
    M, V, n = 3, 20000, 70
    logits, kw = inputs(M, V, 30, BF16, seed=4)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, V, (M, n), generator=g).int()
    ids[0, 5] = -1
    ids[0, 6] = V
    ids[0, 7] = -2 ** 31
    ids[1, 10:40] = 17            # the same token again and again: the last counts
    ids[2, :] = torch.arange(n).flip(0)
    vals = torch.randn(M, n, generator=g) * 10
    vals[2, 3] = -math.inf
    b = dict(bias_ids=ids.to(DEV), bias_values=vals.to(DEV))
    for extra in ({}, kw):
        check(cdna4.process_logits(logits, **b, **extra), *reference(logits, **b, **extra))


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100, 8200, 20011])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_masks(V, dtype):
    g = torch.Generator().manual_seed(V)
    words = (V + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (6, words + 2), generator=g).int()
    mask[0] = -1
    mask[1] = 0                    # a row that may say nothing
    mask[2] = 0
    mask[2, (V - 1) // 32] = int(torch.tensor(1 << ((V - 1) % 32)).int())   # only the last token
    logits, kw = inputs(6, V, 9, dtype, seed=V)
    kw["mask"] = mask.to(DEV)
    out = cdna4.process_logits(logits, **kw)
    check(out, *reference(logits, **kw))
    assert bool((out[1] == -math.inf).all())
    check(cdna4.process_logits(logits, mask=kw["mask"]), *reference(logits, mask=kw["mask"]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logits_of_any_value(dtype):
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    vals = torch.tensor([0.0, -0.0, lo, hi, math.inf, -math.inf, math.nan, torch.finfo(dtype).tiny, 1.0, -1.0]).to(dtype)
    logits = vals.repeat(2, 3).to(DEV)
    V = logits.shape[1]
    kw = dict(history=torch.arange(V).int().repeat(2, 1).to(DEV), repetition=torch.tensor([1.0, 1.5], device=DEV),
              frequency=torch.tensor([0.0, 0.25], device=DEV))
    got = cdna4.process_logits(logits, **kw)
    x, bound = reference(logits, **kw)
    big = x.abs() > torch.finfo(F32).max         # past fp32: infinite there
    x[big] = torch.sign(x[big]) * math.inf
    check(got, x, bound)


def test_strides_and_in_place():
    logits, kw = inputs(5, 777, 40, F32, seed=8)
    wide = torch.full((5, 1000), 3.0, device=DEV)
    wide[:, 100:877] = logits
    view = wide[:, 100:877]
    ref = reference(logits, **kw)
    out = torch.full((5, 900), 7.0, device=DEV)
    cdna4.process_logits(view, out[:, 1:778], **kw)
    check(out[:, 1:778], *ref)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 778:] == 7).all())
    assert cdna4.process_logits(view, view, **kw) is view
    check(view, *ref)
    assert bool((wide[:, :100] == 3).all()) and bool((wide[:, 877:] == 3).all())
    h = logits.to(F16)
    odd = torch.zeros(5, 779, dtype=F16, device=DEV)
    odd[:, 1:778] = h                              # rows start at every alignment
    check(cdna4.process_logits(odd[:, 1:778], **kw), *reference(h, **kw))


def test_same_bits_every_time():
    logits, kw = inputs(8, 32000, 4000, F16, seed=9, hot=200)
    a = cdna4.process_logits(logits, **kw)
    for _ in range(3):
        assert torch.equal(a, cdna4.process_logits(logits, **kw))


def test_other_stream_and_graph():
    logits, kw = inputs(4, 5000, 100, BF16, seed=10, hot=80)
    out = torch.zeros(4, 5000, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    cdna4.process_logits(logits, out, stream=s, **kw)
    s.synchronize()
    check(out, *reference(logits, **kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cdna4.process_logits(logits, out, **kw)
    for seed in (11, 12, 13):
        l2, k2 = inputs(4, 5000, 100, BF16, seed=seed, hot=80)
        logits.copy_(l2)
        for k in kw:
            kw[k].copy_(k2[k])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out, *reference(logits, **kw))


def test_refusals():
    x = torch.zeros(2, 10, device=DEV)
    i = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    f = torch.ones(2, device=DEV)
    for kw in (dict(repetition=f), dict(history=i.long()), dict(history=i, repetition=f.half()), dict(history=i, repetition=f[:1]),
               dict(bias_ids=i), dict(bias_ids=i, bias_values=f), dict(mask=i[:1]), dict(mask=torch.zeros(2, 0, dtype=torch.int32, device=DEV)),
               dict(out=torch.zeros(2, 10, dtype=F16, device=DEV)), dict(out=torch.zeros(2, 9, device=DEV)), dict(history=i.cpu())):
        with pytest.raises((ValueError, cdna4.CDNA4Error)):
            cdna4.process_logits(x, **kw)
    for bad in (x.double(), x[0], x.t()):
        with pytest.raises((ValueError, cdna4.CDNA4Error)):
            cdna4.process_logits(bad)
    assert cdna4.process_logits(torch.zeros(0, 10, device=DEV)).shape == (0, 10)
