"""Paged caches for the tests: pools filled from contiguous keys and values, MXFP4 in 64 bits, references."""
import math

import torch

import cdna4
from serving_util import attend, unit

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def power(e):
    """2^e in float64 for whole numbers e, from its bits: on the GPU a power of two by pow may be a bit off."""
    return (e.long() + 1023 << 52).view(torch.float64)


def quantise(x, dtype):
    """(codes uint8 [..][D], scale bytes [..][D / 32]) of x in 64 bits: the smallest e with max < 7 2^e, nearest codes, ties to even.
    Written for the test alone: the distances to all eight grid values decide."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    lo, hi = (-23, 13) if dtype == torch.float16 else (-125, 125)
    e = torch.full_like(top, lo)
    for step in range(lo, hi):
        e = torch.where(top >= 7 * 2.0 ** step, torch.full_like(e, step + 1), e)
    y = torch.where(bad, torch.zeros_like(b), b / power(e))
    far = (y.abs()[..., None] - GRID.to(x.device)).abs()
    near = far.amin(-1, keepdim=True)
    hit = far == near                                        # two hits at a tie: the even code
    even = torch.tensor([1, 0] * 4, dtype=torch.bool, device=x.device)
    only_even = (hit.sum(-1, keepdim=True) == 2) & even
    code = torch.where(hit.sum(-1, keepdim=True) == 2, only_even & hit, hit).to(torch.uint8).argmax(-1).to(torch.uint8)
    code = code | (torch.signbit(y) & ~bad).to(torch.uint8) << 3
    scale = torch.where(bad, torch.full_like(e, 255), e + 127)[..., 0].to(torch.uint8)
    return code.flatten(-2), scale


def values(code, scale):
    grid = torch.cat([GRID, -GRID]).to(code.device)
    v = grid[code.long()].unflatten(-1, (-1, 32)) * power(scale.long()[..., None] - 127)
    return torch.where(scale[..., None] == 255, torch.full_like(v, float("nan")), v).flatten(-2)


def pack(code, scale, page):
    """[..][page][D] codes and [..][page][D / 32] scales -> [..][page (D / 2 + D / 32)] bytes."""
    return torch.cat([(code[..., ::2] | code[..., 1::2] << 4).flatten(-2), scale.flatten(-2)], -1)


def unpack(pool, page, D):
    split = page * D // 2
    b = pool[..., :split].unflatten(-1, (page, D // 2))
    return torch.stack([b & 15, b >> 4], -1).flatten(-2), pool[..., split:].unflatten(-1, (page, D // 32))


class Paged:
    """Sequences' keys and values [nKVH][n][D] in pages of a pool in random order; rows that hold none are NaN."""

    def __init__(self, lens, HK, D, dtype, page, fmt, seed=0, spare=3, room=2, dev="cuda", scale=1.0):
        self.g = torch.Generator(device=dev)
        self.g.manual_seed(seed)
        rnd = lambda *s: (torch.randn(*s, device=dev, generator=self.g) * scale).to(dtype)
        need = [(n + page - 1) // page for n in lens]
        pages, width = sum(need) + spare, max(need + [1]) + room
        order = torch.randperm(pages, device=dev, generator=self.g).cpu()
        self.free = order[sum(need):].tolist()
        self.tables = torch.full((len(lens), width), -1, dtype=torch.int32)
        self.cache = cdna4.PagedCache(D, HK, page, pages, cdna4.KV_MXFP4 if fmt == "mxfp4" else cdna4.KV_16BIT, width)
        shape = cdna4.paged_pool_shape(self.cache)
        empty = lambda: torch.full(shape, 255, dtype=torch.uint8, device=dev) if fmt == "mxfp4" else torch.full(shape, float("nan"), dtype=dtype, device=dev)
        self.K, self.V = empty(), empty()
        self.k, self.v = [], []                              # what the cache holds, float64
        at = 0
        for b, n in enumerate(lens):
            ids = order[at:at + need[b]]
            at += need[b]
            self.tables[b, :need[b]] = ids.int()
            for pool, held in ((self.K, self.k), (self.V, self.v)):
                x = rnd(HK, n, D)
                if fmt == "mxfp4":
                    code, sc = quantise(x, dtype)
                    x = values(code, sc)
                    for i, p in enumerate(ids.tolist()):
                        c, s = code[:, i * page:(i + 1) * page], sc[:, i * page:(i + 1) * page]
                        r = c.shape[1]
                        pool[p, :, :r * D // 2] = (c[..., ::2] | c[..., 1::2] << 4).flatten(1)
                        pool[p, :, page * D // 2:page * D // 2 + r * D // 32] = s.flatten(1)
                else:
                    for i, p in enumerate(ids.tolist()):
                        r = x[:, i * page:(i + 1) * page]
                        pool[p, :, :r.shape[1]] = r
                held.append(x.double())
        self.tables = self.tables.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)


def attend_two_terms(q, k, v, seen, dtype):
    """(O, bound) as serving_util.attend, for weights that enter the product with V as two 16-bit terms:
      the weights: hi is within u of p, lo within u of p - hi, u^2 in all, or, where lo is below fp16's normal range, half of its
      smallest step, 2^-25, as a part of a sum that is at least 1; over A + |O|, A = sum_j w_j |v_j|;
      scores: as there, (2 D + 16) 2^-24 of sum_d |q_d k_d| / sqrt(D), as a relative error of each weight, twice;
      sums in 32 bits: for 32 keys two matrix instructions, each of them a rounding within and one of the running sum: N / 8, and 16 for
      the joining of parts;
      the output's rounding: half a step of what the rest has left."""
    q, k, v = q.double(), k.double(), v.double()
    N, D = k.shape
    s = ((q @ k.t().contiguous()) / math.sqrt(D)).masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    tot = w.sum(1, keepdim=True)
    w = w / torch.where(tot == 0, torch.ones_like(tot), tot)
    O, A, u, e = w @ v, w @ v.abs(), unit(dtype), 2.0 ** -24
    mag = ((q.abs() @ k.abs().t().contiguous()) / math.sqrt(D)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    off = (u * u + 2 * (2 * D + 16) * e * mag + (N / 8 + 16) * e) * (A + O.abs())
    if dtype == torch.float16:
        off = off + N * 2.0 ** -25 * v.abs().amax(0, keepdim=True)
    return O, off + u * (O.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def decode_reference(q, k, v, dtype, attend=attend):
    """(o, bound) float64 of q [B][nq][HQ][D] over lists of keys and values [HK][n][D]: query i sees all but the last nq - 1 - i."""
    B, nq, HQ, D = q.shape
    O = torch.zeros(B, nq, HQ, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(O)
    for b in range(B):
        HK, n, _ = k[b].shape
        if n == 0:
            continue
        G = HQ // HK
        see = (n - nq + 1 + torch.arange(nq, device=q.device)).repeat_interleave(G)
        seen = torch.arange(n, device=q.device)[None] < see[:, None]
        for h in range(HK):
            x = q[b, :, h * G:(h + 1) * G].reshape(nq * G, D)
            o, e = attend(x, k[b][h], v[b][h], seen, dtype)
            live = (see > 0)[:, None]
            O[b, :, h * G:(h + 1) * G] = torch.where(live, o, torch.zeros_like(o)).view(nq, G, D)
            bound[b, :, h * G:(h + 1) * G] = torch.where(live, e, torch.zeros_like(e)).view(nq, G, D)
    return O, bound


def append_reference(x, w, eps, cos, sin, at):
    """(y, what 32-bit arithmetic and no final rounding may be off by) in float64 of rows x [T][heads][D] normed by w (None: not) and
    rotated by cos, sin[at] (None: not). Roundings of 2^-24: the sum of D squares in a tree of fused steps 12, its mean, eps and square
    root (to 1 ulp) 4, halved by the root, the quotient (2.5 ulp) 5, two products 2: under 18 of each normed value; then the
    product b s 1, the fused sum 1."""
    x = x.double()
    D, e = x.shape[-1], 2.0 ** -24
    off = torch.zeros_like(x)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        off = 18 * e * x.abs()
    if cos is not None:
        c, s = cos.double()[at][:, None], sin.double()[at][:, None]
        swap = lambda t: torch.cat([t[..., D // 2:], t[..., :D // 2]], -1)
        sign = torch.cat([-torch.ones(D // 2), torch.ones(D // 2)]).to(x)
        y = c * x + s * sign * swap(x)
        off = c.abs() * off + s.abs() * swap(off) + e * (s * swap(x)).abs() + e * y.abs()
        x = y
    return x, off
