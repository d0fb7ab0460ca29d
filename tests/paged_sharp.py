"""A bound for the paged attention that a lost or doubled run of positions
breaks, where `paged_cases.Step.reference`'s worst case (every rounding off by
its most, all the same way) lets it pass.

Roundings are independent of one another and each is off by h = half its step
at most, so the error of an output that is a weighted sum of them is
sub-Gaussian with variance sum (weight h)^2 (Hoeffding): past 8 sigma lies less
than 2 exp(-32), and the root mean square over a request's outputs, at least 64
of them, stays below 2 sigma. Which roundings there are, for weights p and
values v = s c + b:

  output            u |o|
  weights (fp16)    u p times what the code term carries, max(|v|, 8 |s|)
  cached v (fp16)   u p |v|
  a score's error e moves o by p e (v - o); e from
    cached k (fp16) scale u sqrt(sum (q k)^2)
    products        2^-16 (fp16 codes as subnormals; fp32 2^-23) times
                    scale sqrt(sum (q ka)^2), ka = |s| c + |b|
    sums            2^-23 sqrt(DH + 16) scale (sqrt(sum (q ka)^2) + |sum q ka|)
    exp2            2^-22
  products with v   2^-16 (fp32 2^-23) p va
  weights below the smallest normal (2^-14 where the largest weight is 2^4 or
                    more): 2^-29 max(p) times 8 max |s|, for each position

and, as additions in the tensor cores truncate, all the same way: 2^-23 for each
of the T / 16 + 16 additions of a run of T positions, times sum p va, and twice
that for the normaliser."""

from __future__ import annotations

import math

import torch

from tests import paged_cases as pc


def parts(s: pc.Step, b: int, hk: int):
    """Request b's positions under cache head hk, cached and then its own (float64):
    k, |s| c + |b| of k, v, |s| c + |b| of v, |s| of v."""
    lo, hi = (int(x) for x in s.cu[b:b + 2])
    n = s.ctx[b]
    blocks = s.tables[b, :pc.cdiv(n, s.page)].long()
    out = []
    for half, new in ((0, s.nk), (1, s.nv)):
        x, mag = s.values(half, b, hk)
        y = new[lo:hi, hk].double()
        sc = s.pools[3 * half + 1][blocks, hk].reshape(len(blocks) * s.page, s.dh // s.group)[:n].double().abs()
        out += [torch.cat([x, y]), torch.cat([mag, y.abs()]),
                torch.cat([sc.repeat_interleave(s.group, 1), torch.zeros_like(y)])]
    k, ka, _, v, va, vs = out
    return k, ka, v, va, vs


def reference(s: pc.Step):
    """(out, sigma, drift), float64 [tokens, H, DH]."""
    n, h, dh = s.q.shape
    half = s.dtype == torch.float16
    u, f = torch.finfo(s.dtype).eps / 2, 2.0 ** -23
    up, fine = (u, 2.0 ** -16) if half else (0.0, f)
    scale = 1 / math.sqrt(dh)
    out = torch.zeros(n, h, dh, dtype=torch.float64, device=s.q.device)
    sigma, drift = torch.zeros_like(out), torch.zeros_like(out)
    cu = s.cu.tolist()
    for b, length in enumerate(s.ctx):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        mask = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=s.q.device).triu(1)
        for hk in range(s.hkv):
            k, ka, v, va, vs = parts(s, b, hk)
            t = k.shape[0]
            cached = torch.arange(t, device=k.device) < length
            for j in range(hk * s.r, (hk + 1) * s.r):
                q = s.q[lo:hi, j].double()
                score = q @ k.T * scale
                score[:, length:].masked_fill_(mask, -math.inf)
                p = torch.softmax(score, -1)
                o = p @ v
                q2 = q * q
                prod = (q2 @ (ka * ka).T).sqrt() * scale
                e2 = (up * scale) ** 2 * (q2 @ (k * k).T) * cached \
                    + (fine * prod) ** 2 \
                    + f * f * (dh + 16) * (prod + (q @ ka.T).abs() * scale) ** 2 + 2.0 ** -44
                w2 = p * p
                carried = torch.maximum(v.abs(), 8 * vs) * cached[:, None] + v.abs() * ~cached[:, None]
                var = (u * o) ** 2 + up * up * (w2 @ (carried ** 2 + v ** 2)) + fine * fine * (w2 @ (va * va))
                pe = w2 * e2
                var += pe @ (v * v) - 2 * o * (pe @ v) + o * o * pe.sum(-1, keepdim=True)
                floor = 2.0 ** -29 * p.amax(-1, keepdim=True) * 8 * torch.maximum(vs.amax(), v.abs().amax() / 8)
                var += floor * floor * t
                out[lo:hi, j], sigma[lo:hi, j] = o, var.clamp(min=0).sqrt()
                drift[lo:hi, j] = f * (t / 16 + 16) * (p @ va + 2 * o.abs()) + torch.finfo(s.dtype).tiny
    return out, sigma, drift


def worst(s: pc.Step, got, ref=None) -> float:
    """How far `got` is from `s`'s outputs, the bound being 1: the farthest element's
    error over 8 sigma + drift, and each request's root mean square error over
    that of 2 sigma + drift. NaN counts as infinitely far."""
    want, sigma, drift = reference(s) if ref is None else ref
    cu, far = s.cu.tolist(), 0.0
    err = (got.double() - want).abs()
    err = torch.where(torch.isfinite(err), err, torch.full_like(err, math.inf))
    for lo, hi in zip(cu, cu[1:]):
        if lo == hi:
            continue
        e, sg, dr = err[lo:hi], sigma[lo:hi], drift[lo:hi]
        rms = [float(x.square().mean().sqrt()) for x in (e, 2 * sg + dr)]
        far = max(far, float((e / (8 * sg + dr)).max()), rms[0] / rms[1])
    return far


def check(s: pc.Step, got, ref=None) -> float:
    assert got.dtype == s.dtype and tuple(got.shape) == tuple(s.q.shape)
    far = worst(s, got, ref)
    assert far <= 1.0, f"error is {far:.3g} of its bound"
    return far


# ---- steps in which every block of positions shows -------------------------------
def mark(s: pc.Step, blocks) -> None:
    """Half of the weight on one block of 16 cached positions of each (request,
    cache head), and values nowhere else, the step's own among them: the block
    lost leaves 0 of it, doubled 4/3 of it. blocks[b][hk] is the block's number.
    Queries and keys are constant along DH (keys 0 outside the block)."""
    s.q.fill_(1.0)
    s.nk.fill_(0.0)
    s.nv.fill_(0.0)
    for t in s.pools[1], s.pools[2], s.pools[4], s.pools[5]:
        t.zero_()                                  # free rows too: they are not read
    for b, n in enumerate(s.ctx):
        for hk in range(s.hkv):
            first = 16 * blocks[b][hk]
            held = min(16, n - first)
            # scores sqrt(DH) k in the block, 0 elsewhere, own entries included
            # (as many as the last token sees)
            k = math.log(max(n - held + s.new[b], 1) / held) / math.sqrt(s.dh)
            rows = torch.arange(first, first + held, device=s.tables.device)
            at = s.tables[b, rows // s.page].long()
            s.pools[2][at, hk, rows % s.page] = k
            s.pools[4][at, hk, rows % s.page] = 1 / 16
            s.pools[5][at, hk, rows % s.page] = 0.5


def without(s: pc.Step, b: int, first: int, last: int, times: int = 0):
    """The 64-bit outputs with request b's cached positions first .. last - 1 taken
    `times` times, in s's dtype: what a kernel that lost or doubled them gives."""
    want = reference(s)[0].clone()
    lo, hi = (int(x) for x in s.cu[b:b + 2])
    mask = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=s.q.device).triu(1)
    for hk in range(s.hkv):
        k, _, v, _, _ = parts(s, b, hk)
        for j in range(hk * s.r, (hk + 1) * s.r):
            score = s.q[lo:hi, j].double() @ k.T / math.sqrt(s.dh)
            score[:, s.ctx[b]:].masked_fill_(mask, -math.inf)
            score[:, first:last] += math.log(times) if times else -math.inf
            want[lo:hi, j] = torch.softmax(score, -1) @ v
    return want.to(s.dtype)


def outlier(s: pc.Step, b: int, hk: int, pos: int) -> None:
    """Request b's position `pos` under cache head hk: scales of V 2^13 times what
    they were, and values that are 0 in every second dim, there with the code 8."""
    page, row = s.tables[b, pos // s.page], pos % s.page
    s.pools[4][page, hk, row] *= 2.0 ** 13
    s.pools[5][page, hk, row] = -8 * s.pools[4][page, hk, row]
    w = s.pools[3][page, hk, row]
    s.pools[3][page, hk, row] = (w & 0x70707070) | 0x08080808
