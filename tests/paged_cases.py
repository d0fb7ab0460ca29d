"""Plain 64-bit implementations of the paged cache's operators, the cases they
are run on, and the error bounds of the kernels' arithmetic."""

from __future__ import annotations

import math
import random

import numpy as np
import torch

from oracle import quant

DEV = "cuda"


def cdiv(a, b):
    return -(-a // b)


# ---- tables -----------------------------------------------------------------
def tables_reference(lens, new, tables, free, n_free, page, max_tokens):
    """build_tables, request by request on Python integers."""
    lens, new = [max(x, 0) for x in lens], [max(x, 0) for x in new]
    tables = [list(r) for r in tables]
    width = len(tables[0])
    lack = [cdiv(a + n, page) - cdiv(a, page) for a, n in zip(lens, new)]
    status = (sum(lack) > n_free) * 1 + any(cdiv(a + n, page) > width for a, n in zip(lens, new)) * 2 \
        + (sum(new) > max_tokens) * 4
    if status:
        return ([0] * (len(lens) + 1), [-1] * max_tokens, [0] * max_tokens, lens, n_free, status, tables)
    cu, slots, positions, top = [0], [], [], n_free
    for b, (a, n) in enumerate(zip(lens, new)):
        for c in range(cdiv(a, page), cdiv(a + n, page)):
            top -= 1
            tables[b][c] = free[top]
        for p in range(a, a + n):
            slots.append(tables[b][p // page] * page + p % page)
            positions.append(p)
        cu.append(cu[-1] + n)
    pad = max_tokens - len(slots)
    return (cu, slots + [-1] * pad, positions + [0] * pad, [a + n for a, n in zip(lens, new)], top, 0, tables)


def truncate_reference(lens, keep, tables, free, n_free, page):
    lens = [max(x, 0) for x in lens]
    keep = [min(a, max(k, 0)) for a, k in zip(lens, keep)]
    free = list(free)
    for b, (a, k) in enumerate(zip(lens, keep)):
        for c in range(cdiv(k, page), cdiv(a, page)):
            free[n_free] = tables[b][c]
            n_free += 1
    return keep, n_free, free


# ---- attention ----------------------------------------------------------------
class Step:
    """The inputs of one attention step; `ctx` and `new` per request. Cached
    values are quantized by the oracle; rows the step may not read (past each
    length, free pages) hold NaN scales and biases."""

    def __init__(self, ctx, new, hkv, r, dh, group, page, dtype, seed=0, pad=0, spread=1.0, packed=True,
                 extra_width=0):
        self.ctx, self.new, self.hkv, self.r, self.dh, self.group, self.page = ctx, new, hkv, r, dh, group, page
        self.dtype = dtype
        rng = np.random.default_rng(seed)
        npdt = np.float16 if dtype == torch.float16 else np.float32
        need = [cdiv(c, page) for c in ctx]
        pages = sum(need) + 2
        order = rng.permutation(pages)
        width = max([1] + need) + extra_width
        tables = np.full((len(ctx), width), -7, np.int32)
        self.pools = []
        rows = []                                  # (slot) of every cached position, in request order
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = order[at:at + n]
            at += n
            rows += [int(tables[b, p // page]) * page + p % page for p in range(ctx[b])]
        rows = np.array(rows, np.int64)
        for _ in range(2):
            x = (rng.standard_normal((len(rows), hkv, dh)) * rng.uniform(0.2, 2.0, dh) * spread
                 + rng.standard_normal(dh) * 0.3).astype(npdt)
            words = rng.integers(0, 1 << 32, (pages, hkv, page, dh // 8), dtype=np.uint64).astype(np.uint32)
            scales = np.full((pages, hkv, page, dh // group), np.nan, npdt)
            biases = scales.copy()
            if len(rows):
                codes, s, z = quant.canonical_quantize(x.reshape(-1, dh), 4, group)
                w = quant.pack_codes(codes, 4).reshape(len(rows), hkv, -1)
                words[rows // page, :, rows % page] = w
                scales[rows // page, :, rows % page] = s.reshape(len(rows), hkv, -1)
                biases[rows // page, :, rows % page] = z.reshape(len(rows), hkv, -1)
            self.pools += [torch.from_numpy(words.view(np.int32)).to(DEV), torch.from_numpy(scales).to(DEV),
                           torch.from_numpy(biases).to(DEV)]
        n = sum(new) + pad
        h = hkv * r
        g = torch.Generator().manual_seed(seed + 1)
        qkv = (torch.randn(n, h + 2 * hkv, dh, generator=g) * spread).to(dtype).to(DEV)
        self.q, self.nk, self.nv = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        if not packed:
            self.q, self.nk, self.nv = (x.contiguous() for x in (self.q, self.nk, self.nv))
        self.tables = torch.from_numpy(tables).to(DEV)
        self.ctx_t = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)

    def call(self, paged, **over):
        kw = dict(block_tables=self.tables, ctx_lens=self.ctx_t, cu_new=self.cu, max_new=max(self.new),
                  max_ctx=max(self.ctx))
        kw.update(over)
        return paged.attend(self.q, *self.pools, self.nk, self.nv, **kw)

    def values(self, half, b, hk):
        """(values [ctx, DH], |scale| * code + |bias|) of request b in float64."""
        w, s, z = self.pools[3 * half:3 * half + 3]
        blocks = self.tables[b, :cdiv(self.ctx[b], self.page)].long()
        n = self.ctx[b]
        w, s, z = (x[blocks, hk].reshape(len(blocks) * self.page, x.shape[-1])[:n] for x in (w, s, z))
        w, s, z = w.long() & 0xFFFFFFFF, s.double(), z.double()
        codes = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], -1).reshape(n, self.dh).double()
        s, z = (x.repeat_interleave(self.group, 1) for x in (s, z))
        return s * codes + z, s.abs() * codes + z.abs()

    def reference(self):
        """(out float64, error bound), both [tokens, H, DH].

        The bound counts, relative to A = sum_j p_j |v_j| (and |o| for the
        output): the output's rounding u; for float16, P, V and K each rounded
        to float16 once (u each; K's reaches a score as e_j = scale * u * sum
        |q k_j|, a weight as e_j relatively, and the normaliser again: 2 max
        e_j); and float32 arithmetic everywhere, dots of DH terms and sums of T
        weights accumulated term by term, each addition off by 2^-23 at most
        (tensor cores may truncate), with codes times scale and bias apart,
        whose magnitudes are |scale| c + |bias|."""
        n, h, dh = self.q.shape
        u = torch.finfo(self.dtype).eps / 2
        f = 2.0 ** -23
        half = self.dtype == torch.float16
        out = torch.zeros(n, h, dh, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        scale = 1 / math.sqrt(dh)
        cu = self.cu.tolist()
        for b, length in enumerate(self.ctx):
            lo, hi = cu[b], cu[b + 1]
            if lo == hi:
                continue
            mask = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=DEV).triu(1)
            for hk in range(self.hkv):
                k, ka = self.values(0, b, hk)
                v, va = self.values(1, b, hk)
                nk, nv = self.nk[lo:hi, hk].double(), self.nv[lo:hi, hk].double()
                k, ka, v, va = (torch.cat([x, y]) for x, y in ((k, nk), (ka, nk.abs()), (v, nv), (va, nv.abs())))
                for j in range(hk * self.r, (hk + 1) * self.r):
                    q = self.q[lo:hi, j].double()
                    s = q @ k.T * scale
                    mag = q.abs() @ ka.T * scale
                    e = (q.abs() @ k.abs().T * scale * u if half else 0) + mag * f * (dh + 8)
                    s[:, length:].masked_fill_(mask, -math.inf)
                    e = torch.where(torch.isinf(s), torch.zeros_like(e), e)
                    p = torch.softmax(s, -1)
                    o = p @ v
                    a = p @ va
                    rel = (2 * u if half else 0) + f * (v.shape[0] + 16) + 2 * e.amax(-1, keepdim=True)
                    out[lo:hi, j] = o
                    tol[lo:hi, j] = u * o.abs() + a * rel + torch.finfo(self.dtype).tiny
        return out, tol

    def check(self, got):
        want, tol = self.reference()
        n = sum(self.new)
        assert got.dtype == self.dtype and tuple(got.shape) == tuple(self.q.shape)
        err = (got[:n].double() - want[:n]).abs()
        worst = float((err / tol[:n]).max()) if n else 0.0
        assert worst <= 1.0 and bool(torch.isfinite(got[:n]).all()), f"error is {worst:.3g} of its bound"
        return worst


def log_lengths(rng: random.Random, n, lo, hi):
    return [min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1)))))) for _ in range(n)]
