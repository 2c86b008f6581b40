"""64-bit references and derived error bounds of the batched attention operators' tests."""
import math

import torch

DEV = torch.device("cuda", 0)


def unit(dtype):
    """Half a step of a 16-bit type, relative to the value."""
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, seen, dtype):
    """(O, bound) in float64 for one head: q [n][D], k, v [N][D], seen bool [n][N]. bound is what a kernel with
    16-bit weights, 32-bit sums and a 16-bit output may be off by, per element:
      the weights' rounding: u sum_j w_j |v_j - O| <= u (A + |O|), A = sum_j w_j |v_j|;
      fp16 weights below 2^-14 of the largest: 2^-25 each, as a part of a sum that is at least 1;
      scores: D + 8 roundings of 2^-24 of sum_d |q_d k_d| / sqrt(D), and as many of |s| again for the scaling and the
      exponent, as a relative error of each weight, twice (numerator and denominator), over A + |O|;
      the 32-bit sums over N keys: 2^-24 sqrt-free worst case N 2^-24 is not reached by tree sums of at most 32
      keys per matrix instruction: N / 16 + 16 roundings;
      the output's rounding: u |O|, and the type's smallest step below its normal range."""
    q, k, v = q.double(), k.double(), v.double()
    n, D = q.shape
    N = k.shape[0]
    if N == 0:
        z = torch.zeros(n, D, dtype=torch.float64, device=q.device)
        return z, z.clone()
    s = (q @ k.t().contiguous()) / math.sqrt(D)
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    tot = w.sum(1, keepdim=True)
    w = w / torch.where(tot == 0, torch.ones_like(tot), tot)
    O = w @ v
    A = w @ v.abs()
    u = unit(dtype)
    mag = (q.abs() @ k.abs().t().contiguous()) / math.sqrt(D)
    mag = mag.masked_fill(~seen, 0.0).amax(1, keepdim=True)
    e = 2.0 ** -24
    rel = 2 * (2 * D + 16) * e * mag + (N / 16 + 16) * e
    bound = (u + rel) * (A + O.abs()) + u * O.abs()
    if dtype == torch.float16:
        bound = bound + N * 2.0 ** -25 * v.abs().amax(0, keepdim=True) + 2.0 ** -25
    return O, bound


def packed_reference(Q, K, V, cu, D, G, dtype, Kp=None, Vp=None, P=0):
    """(O, bound, covered rows) for packed prompts; cu a host list."""
    T, HQ = Q.shape[0], Q.shape[1]
    O = torch.zeros(T, HQ, D, dtype=torch.float64, device=Q.device)
    bound = torch.zeros_like(O)
    covered = torch.zeros(T, dtype=torch.bool, device=Q.device)
    for s in range(len(cu) - 1):
        a, b = cu[s], cu[s + 1]
        if b <= a:
            continue
        covered[a:b] = True
        seen = torch.ones(b - a, P + b - a, dtype=torch.bool, device=Q.device).tril(P)
        for h in range(HQ):
            k, v = K[a:b, h // G], V[a:b, h // G]
            if P:
                k, v = torch.cat([Kp[h // G, :P], k]), torch.cat([Vp[h // G, :P], v])
            O[a:b, h], bound[a:b, h] = attend(Q[a:b, h], k, v, seen, dtype)
    return O, bound, covered


def check(got, ref, bound, what=""):
    d = (got.double() - ref).abs()
    ok = d <= bound
    worst = float((d / bound.clamp(min=1e-30)).max()) if d.numel() else 0.0
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {d.numel()} outside the bound, worst {worst:.3g} of it"
    return worst


def cu_of(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def shared_reference(q, Kp, Vp, K, V, lens, G, dtype, P=0):
    """(o, bound) of one query per sequence; lens a host list."""
    B, HQ, D = q.shape
    O = torch.zeros(B, HQ, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(O)
    for b in range(B):
        for h in range(HQ // G):
            k, v = [], []
            if P:
                k.append(Kp[h, :P]), v.append(Vp[h, :P])
            if lens is not None and lens[b] > 0:
                k.append(K[b, h, :lens[b]]), v.append(V[b, h, :lens[b]])
            if not k:
                continue
            k, v = torch.cat(k), torch.cat(v)
            sl = slice(h * G, (h + 1) * G)
            O[b, sl], bound[b, sl] = attend(q[b, sl], k, v, torch.ones(G, k.shape[0], dtype=torch.bool, device=q.device), dtype)
    return O, bound
