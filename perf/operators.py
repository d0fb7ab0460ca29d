"""The operators of a paged 4-bit K/V cache, as they are timed.

Four operators carry a serving step over a cache that is held in pages:

* grow   -- block tables, token slots, positions and offsets of a step, built
            on the GPU from the requests' lengths and a stack of free pages;
* trim   -- requests cut back to a kept length (a rejected draft, a finished
            request), their pages pushed back on the stack;
* append -- the step's keys and values quantized to 4 bits into their slots,
            and read back from the cache as the values it then holds;
* attend -- attention of the step's tokens over their cached positions (4-bit
            codes with a scale and a bias per group) and over the step's own
            keys and values, which enter at full precision, causally.

Sizes follow this repository's decode shapes: 32 query heads over 8 cache
heads of 128, 64 over 8 for one long sequence, groups of 64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _tables_case(kind, rows, page, len_lo, len_hi, step_lo, step_hi, pad):
    return {"kind": kind, "rows": rows, "page": page, "len_lo": len_lo, "len_hi": len_hi,
            "step_lo": step_lo, "step_hi": step_hi, "pad": pad}


def _append_case(tokens, dtype, kv_heads, head_dim, group, page, pad):
    return {"kind": "append", "tokens": tokens, "dtype": dtype, "kv_heads": kv_heads,
            "head_dim": head_dim, "group": group, "page": page, "pad": pad}


def _attend_case(rows, ctx_lo, ctx_hi, new_lo, new_hi, singles, dtype, kv_heads, share, head_dim,
                 group, page):
    """`singles` of the `rows` requests bring one token, the others new_lo..new_hi."""
    return {"kind": "attend", "rows": rows, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "new_lo": new_lo,
            "new_hi": new_hi, "singles": singles, "dtype": dtype, "kv_heads": kv_heads,
            "share": share, "head_dim": head_dim, "group": group, "page": page}


def listed():
    return [
        # one decode step of a batch of 32: one token each, a page now and then
        {"name": "grow decode 32", **_tables_case("grow", 32, 64, 512, 8192, 1, 1, 0)},
        # a batch of 512 with prompts of up to 1000 tokens admitted, padded for a captured step
        {"name": "grow prompts 512", **_tables_case("grow", 512, 16, 0, 4000, 1, 1000, 97)},
        # rejected drafts: 32 requests give back up to 7 tokens
        {"name": "trim drafts 32", **_tables_case("trim", 32, 16, 512, 8192, 1, 7, 0)},
        # a batch that has ended: 512 requests give back all they hold
        {"name": "trim ended 512", **_tables_case("trim", 512, 16, 1, 8192, 8192, 8192, 0)},
        # the appended tokens of one decode step, some rows of the batch unused
        {"name": "append decode 32", **_append_case(32, "float16", 8, 128, 64, 64, 3)},
        # a chunk of prompts
        {"name": "append chunk 8192", **_append_case(8192, "float16", 8, 128, 64, 64, 0)},
        # the smallest step: one sequence behind a short prompt
        {"name": "attend 1x512", **_attend_case(1, 512, 512, 1, 1, 1, "float16", 8, 4, 128, 64, 64)},
        # a decode batch of long sequences
        {"name": "attend 32x8192", **_attend_case(32, 8192, 8192, 1, 1, 32, "float16", 8, 4, 128, 64, 64)},
        # one very long sequence, many query heads
        {"name": "attend 1x131072", **_attend_case(1, 131072, 131072, 1, 1, 1, "float16", 8, 8, 128, 64, 64)},
        # drafts verified in float32, heads of 64, small groups and pages, odd lengths
        {"name": "attend drafts float32", **_attend_case(9, 37, 3001, 2, 5, 2, "float32", 4, 3, 64, 32, 16)},
        # a chunk of 4096 tokens of one long prompt
        {"name": "attend chunk 4096", **_attend_case(1, 8192, 8192, 4096, 4096, 0, "float16", 8, 4, 128, 64, 64)},
        # decoding requests and prompts of odd lengths in one step, an empty context among them
        {"name": "attend mixed 16", **_attend_case(16, 0, 4001, 65, 777, 12, "float16", 8, 4, 128, 64, 16)},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm (from 1, where lo is 0)."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def _attend_cost(case):
    """(bytes read of the cache, operations, largest tensor of the plain form)."""
    ctx, new = _attend_lengths(case)
    heads = case["kv_heads"] * case["share"]
    flops = sum(4.0 * case["head_dim"] * heads * n * (c + (n + 1) / 2) for c, n in zip(ctx, new))
    top_c, top_n = max(ctx), max(new)
    plain = 4.0 * case["rows"] * max(heads * top_n * (top_c + top_n),
                                     case["kv_heads"] * top_c * case["head_dim"])
    return sum(ctx) * case["kv_heads"] * case["head_dim"], flops, plain


def draw(rng):
    kind = rng.choice(["grow", "trim", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if kind in ("grow", "trim"):
        rows = _log(rng, 1, 512)
        len_hi = _log(rng, 1, 8192)
        step_hi = _log(rng, 1, 1000) if kind == "grow" else _log(rng, 1, 8192)
        return _tables_case(kind, rows, page, _log(rng, 0, len_hi), len_hi, _log(rng, 1, step_hi),
                            step_hi, rng.choice([0, 0, rng.randint(1, 200)]))
    head_dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 64, 128) if g <= head_dim])
    kv_heads = rng.choice([1, 2, 4, 8])
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        return _append_case(tokens, rng.choice(["float16", "float16", "float32"]), kv_heads,
                            head_dim, group, page, rng.choice([0, 0, _log(rng, 1, 100)]))
    while True:
        form = rng.choice(["decode", "decode", "drafts", "chunk", "mixed"])
        rows = _log(rng, 1, 64)
        ctx_hi = _log(rng, 1, 131072)
        ctx_lo = _log(rng, 0, ctx_hi)
        share = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        dtype = "float16"
        singles, new_lo, new_hi = rows, 1, 1
        if form == "drafts":
            singles, new_lo, new_hi = 0, 1, rng.randint(2, 8)
        elif form in ("chunk", "mixed"):
            singles = 0 if form == "chunk" else rng.randint(1, rows)
            new_hi = _log(rng, 9, 4096)
            new_lo = _log(rng, 9, new_hi)
        if form in ("decode", "drafts") and rng.random() < 0.25:
            dtype = "float32"
        case = _attend_case(rows, ctx_lo, ctx_hi, new_lo, new_hi, singles, dtype, kv_heads, share,
                            head_dim, group, page)
        read, flops, plain = _attend_cost(case)
        if read <= 32 * 8192 * 8 * 128 and flops <= 6e11 and plain <= 7e9:
            return case


def _attend_lengths(case):
    """(cached lengths, new tokens) of each request: a property of the case."""
    rng = random.Random("attend %d %d %d %d" % (case["rows"], case["ctx_hi"], case["new_hi"], case["singles"]))
    least = case["ctx_lo"] or min(256, case["ctx_hi"])
    ctx = [_log(rng, least, case["ctx_hi"]) for _ in range(case["rows"])]
    new = [1] * case["singles"] + [_log(rng, case["new_lo"], case["new_hi"])
                                   for _ in range(case["rows"] - case["singles"])]
    rng.shuffle(new)
    ctx[rng.randrange(case["rows"])] = case["ctx_hi"]
    if case["ctx_lo"] == 0:
        ctx[new.index(max(new))] = 0
    return ctx, new


def _tables_lengths(case):
    """(lengths held, tokens to add or to give back) of each request."""
    rng = random.Random("tables %d %d %d" % (case["rows"], case["len_hi"], case["step_hi"]))
    held = [_log(rng, case["len_lo"], case["len_hi"]) for _ in range(case["rows"])]
    step = [_log(rng, case["step_lo"], case["step_hi"]) for _ in range(case["rows"])]
    return held, step


def _pages(n, page):
    return -(-n // page)


def work(case):
    if case["kind"] in ("grow", "trim"):
        held, step = _tables_lengths(case)
        rows = case["rows"]
        if case["kind"] == "grow":
            tokens = sum(step)
            fresh = sum(_pages(h + s, case["page"]) - _pages(h, case["page"]) for h, s in zip(held, step))
            # lengths and steps in; offsets, lengths, slots (8 bytes), positions out; free ids moved
            return {"bytes": 16 * rows + 12 * (tokens + case["pad"]) + 8 * fresh + 12, "flops": 0}
        back = sum(_pages(h, case["page"]) - _pages(max(h - s, 0), case["page"]) for h, s in zip(held, step))
        return {"bytes": 12 * rows + 8 * back + 8, "flops": 0}
    size = 2 if case["dtype"] == "float16" else 4
    packed = case["head_dim"] // 2 + 2 * size * (case["head_dim"] // case["group"])
    if case["kind"] == "append":
        rows = 2 * case["tokens"] * case["kv_heads"]
        # read, written packed, read packed, written as values
        return {"bytes": rows * (2 * case["head_dim"] * size + 2 * packed) + 8 * case["tokens"], "flops": 0}
    ctx, new = _attend_lengths(case)
    heads = case["kv_heads"] * case["share"]
    own_rows = sum(new) * case["head_dim"] * size * (2 * heads + 2 * case["kv_heads"])
    return {"bytes": sum(ctx) * case["kv_heads"] * 2 * packed + own_rows
            + 4 * sum(_pages(c, case["page"]) for c in ctx), "flops": _attend_cost(case)[1]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table_of(lengths, page, width, order, device):
    """Block tables [rows, width]: each request's pages are the next ones of
    `order`; entries behind them are -1. Returns (tables, pages used)."""
    need = torch.tensor([_pages(n, page) for n in lengths], device=device)
    off = need.cumsum(0) - need
    col = torch.arange(width, device=device)
    at = (off[:, None] + col).clamp(max=order.numel() - 1)
    tables = torch.where(col < need[:, None], order[at], torch.full_like(at, -1, dtype=order.dtype))
    return tables.to(torch.int32).contiguous(), int(need.sum())


def _kv_values(gen, rows, head_dim, dtype):
    """Keys or values as projections leave them: normal, with a few strong
    channels and an offset per channel."""
    gain = 0.5 + torch.rand(head_dim, generator=gen, device="cuda")
    gain[:: max(1, head_dim // 4)] *= 4.0
    shift = 0.3 * torch.randn(head_dim, generator=gen, device="cuda")
    x = torch.randn(rows, head_dim, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(gain).add_(shift).to(dtype)


def _pool(gen, pages, kv_heads, page, head_dim, group, dtype):
    """One packed pool (words, scales, biases), filled with quantized values."""
    rows = pages * kv_heads * page
    chunk = 1 << 19
    parts = [_plain_quantize(_kv_values(gen, min(chunk, rows - r), head_dim, dtype), group)
             for r in range(0, rows, chunk)]
    lead = (pages, kv_heads, page)
    return [torch.cat(p).reshape(lead + (-1,)) for p in zip(*parts)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    page = case["page"]
    s = {"kind": case["kind"], "page": page}
    if case["kind"] in ("grow", "trim"):
        held, step = _tables_lengths(case)
        longest = max(h + x for h, x in zip(held, step)) if case["kind"] == "grow" else max(held)
        width = _pages(longest, page) + 2
        total = sum(_pages(h, page) for h in held)
        fresh = sum(_pages(h + x, page) for h, x in zip(held, step)) - total if case["kind"] == "grow" else 0
        pool = total + fresh + 37
        order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
        tables, used = _table_of(held, page, width, order, "cuda")
        free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        free[:pool - used] = order[used:]
        s.update(tables=tables, free=free, n_free=_ints([pool - used]), lens=_ints(held))
        if case["kind"] == "grow":
            s.update(new=_ints(step), max_tokens=sum(step) + case["pad"])
        else:
            s.update(keep=_ints([max(h - x, 0) for h, x in zip(held, step)]))
        return s
    dtype = DTYPES[case["dtype"]]
    hkv, dh, group = case["kv_heads"], case["head_dim"], case["group"]
    if case["kind"] == "append":
        n = case["tokens"]
        pages = _pages(n, page) * 2 + 1
        s["k"] = _pool(gen, pages, hkv, page, dh, group, dtype)
        s["v"] = _pool(gen, pages, hkv, page, dh, group, dtype)
        # the step's tokens fill runs of whole pages and one part, in the pool's order
        order = torch.randperm(pages, generator=gen, device="cuda")
        tok = torch.arange(n, device="cuda") + 5
        slots = order[tok // page] * page + tok % page
        s["slots"] = torch.cat([slots, torch.full((case["pad"],), -1, device="cuda", dtype=torch.int64)])
        n += case["pad"]
        s["padded"] = bool(case["pad"])
        # keys and values come out of one projection, beside the queries
        qkv = _kv_values(gen, n * 3 * hkv, dh, dtype).view(n, 3 * hkv, dh)
        s["new_k"], s["new_v"] = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:]
        return s
    ctx, new = _attend_lengths(case)
    heads = hkv * case["share"]
    used = sum(_pages(c, page) for c in ctx)
    pages = used + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    width = max(1, _pages(max(ctx), page))
    s["tables"], _ = _table_of(ctx, page, width, order, "cuda")
    s["k"] = _pool(gen, pages, hkv, page, dh, group, dtype)
    s["v"] = _pool(gen, pages, hkv, page, dh, group, dtype)
    n = sum(new)
    qkv = torch.empty(n, heads + 2 * hkv, dh, dtype=dtype, device="cuda")
    qkv[:, :heads] = torch.randn(n, heads, dh, generator=gen, device="cuda").to(dtype)
    for at in (heads, heads + hkv):
        qkv[:, at:at + hkv] = _kv_values(gen, n * hkv, dh, dtype).view(n, hkv, dh)
    s["q"], s["new_k"], s["new_v"] = qkv[:, :heads], qkv[:, heads:heads + hkv], qkv[:, heads + hkv:]
    s["ctx"] = _ints(ctx)
    s["cu"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
    s["max_ctx"], s["max_new"] = max(ctx), max(new)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _round_half_away(x):
    return torch.sign(x) * torch.floor(torch.abs(x) + 0.5)


def _plain_quantize(x, group):
    """x [rows, DH] -> (words int32 [rows, DH/8], scales, biases [rows, DH/group]):
    the affine 4-bit quantizer, every step rounded in float32."""
    rows, dh = x.shape
    g = x.float().reshape(rows, dh // group, group)
    lo = g.amin(2)
    hi = g.amax(2).clamp(min=0.0)
    step = ((hi - lo) / torch.full_like(hi, 15.0)).clamp(min=1e-7)
    low_side = lo.abs() > hi.abs()
    step = torch.where(low_side, step, -step)
    edge = torch.where(low_side, lo, hi)
    n_edge = _round_half_away(edge / step)
    flat = n_edge == 0
    step = torch.where(flat, step, edge / torch.where(flat, torch.ones_like(n_edge), n_edge))
    bias = torch.where(flat, torch.zeros_like(edge), edge)
    codes = _round_half_away((g - bias[..., None]) / step[..., None]).clamp(max=15.0).to(torch.int32)
    codes = codes.reshape(rows, dh // 8, 8)
    shift = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    words = (codes << shift).sum(-1, dtype=torch.int32)
    return words, step.to(x.dtype), bias.to(x.dtype)


def _plain_values(words, scales, biases):
    """Packed rows [..., W] as float32 values [..., 8 W]."""
    shift = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    codes = ((words[..., None] >> shift) & 15).float()
    lead, dh = words.shape[:-1], words.shape[-1] * 8
    codes = codes.reshape(lead + (scales.shape[-1], -1))
    return (codes * scales.float()[..., None] + biases.float()[..., None]).reshape(lead + (dh,))


def _plain_grow(s):
    page, tables, free = s["page"], s["tables"], s["free"]
    lens, new = s["lens"].long().clamp(min=0), s["new"].long().clamp(min=0)
    rows, width = tables.shape
    have = (lens + page - 1) // page
    need = (lens + new + page - 1) // page
    n_free = s["n_free"].long()
    status = ((need - have).sum() > n_free).int() + 2 * (need > width).any().int() \
        + 4 * (new.sum() > s["max_tokens"]).int()
    new = torch.where(status == 0, new, torch.zeros_like(new))
    need = torch.where(status == 0, need, have)
    fresh = need - have
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    first = fresh.cumsum(0) - fresh
    col = torch.arange(width, device=tables.device)
    at = n_free - 1 - (first[:, None] + col - have[:, None])
    took = (col >= have[:, None]) & (col < need[:, None])
    tables.copy_(torch.where(took, free[at.clamp(0, free.numel() - 1)], tables))
    tok = torch.arange(s["max_tokens"], device=tables.device)
    row = torch.searchsorted(cu[1:], tok, right=True).clamp(max=rows - 1)
    pos = lens[row] + tok - cu[row]
    live = tok < cu[-1]
    held = tables[row, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(live, held * page + pos % page, torch.full_like(pos, -1))
    return {"cu_new": cu.int(), "slots": slots, "positions": torch.where(live, pos, torch.zeros_like(pos)).int(),
            "lens": (lens + new).int(), "n_free": (n_free - fresh.sum()).int(),
            "status": status.reshape(1).int(), "tables": tables}


def _plain_trim(s):
    page, tables, free = s["page"], s["tables"], s["free"]
    lens = s["lens"].long().clamp(min=0)
    keep = torch.minimum(lens, s["keep"].long().clamp(min=0))
    kept = (keep + page - 1) // page
    back = (lens + page - 1) // page - kept
    ends = back.cumsum(0)
    n_free = s["n_free"].long()
    e = torch.arange(free.numel(), device=free.device) - n_free
    row = torch.searchsorted(ends, e, right=True).clamp(max=lens.numel() - 1)
    col = (kept[row] + e - (ends[row] - back[row])).clamp(0, tables.shape[1] - 1)
    live = (e >= 0) & (e < ends[-1])
    free.copy_(torch.where(live, tables[row, col], free))
    return {"lens": keep.int(), "n_free": (n_free + ends[-1]).clamp(max=free.numel()).int(), "free": free}


def _plain_append(s):
    page, slots = s["page"], s["slots"]
    hkv, dh = s["new_k"].shape[1:]
    out = []
    for pool, x in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        at, y = slots, x
        if s["padded"]:
            at, y = slots[slots >= 0], x[slots >= 0]
        group = dh // pool[1].shape[-1]
        rows = _plain_quantize(y.reshape(-1, dh), group)
        block, off = at // page, at % page
        for p, r in zip(pool, rows):
            p[block, :, off] = r.view(-1, hkv, p.shape[-1])
        back = slots.clamp(min=0)
        got = _plain_values(*[p[back // page, :, back % page] for p in pool])
        out.append(torch.where((slots >= 0)[:, None, None], got, torch.zeros_like(got)).to(x.dtype))
    return out


def _plain_attend(s):
    q, page = s["q"], s["page"]
    n, heads, dh = q.shape
    hkv = s["new_k"].shape[1]
    ctx, cu = s["ctx"].long(), s["cu"].long()
    rows, top = ctx.numel(), s["max_new"]
    scale = dh ** -0.5
    tok = cu[:-1, None] + torch.arange(top, device=q.device)
    live = tok < cu[1:, None]                                      # [B, L]
    tok = tok.clamp(max=n - 1)
    qf = q[tok].float().view(rows, top, hkv, -1, dh).permute(0, 2, 3, 1, 4).reshape(rows, hkv, -1, dh)
    share = heads // hkv
    nk, nv = (x[tok].float().permute(0, 2, 1, 3) for x in (s["new_k"], s["new_v"]))
    order = torch.arange(top, device=q.device)
    seen = (order[None, :] <= order[:, None]) & live[:, None, :]    # [B, L, L]
    own_scores = (qf @ nk.transpose(2, 3)).mul_(scale).view(rows, hkv, share, top, top)
    own_scores.masked_fill_(~seen[:, None, None], -math.inf)
    own_scores = own_scores.view(rows, hkv, share * top, top)
    blocks = s["tables"][:, :_pages(s["max_ctx"], page)].long().clamp(min=0)
    if blocks.shape[1] == 0:
        p = torch.exp(own_scores - own_scores.amax(-1, keepdim=True))
        o = (p @ nv) / p.sum(-1, keepdim=True)
    else:
        past = torch.arange(blocks.shape[1] * page, device=q.device) < ctx[:, None]
        kk, vv = (_plain_values(*[p[blocks] for p in s[x]]).transpose(1, 2).reshape(rows, hkv, -1, dh)
                  for x in ("k", "v"))
        scores = (qf @ kk.transpose(2, 3)).mul_(scale)
        del kk
        scores.masked_fill_(~past[:, None, None], -math.inf)
        top_score = torch.maximum(scores.amax(-1, keepdim=True), own_scores.amax(-1, keepdim=True))
        top_score = top_score.clamp(min=-1e30)
        p = scores.sub_(top_score).exp_()
        p_own = torch.exp(own_scores - top_score)
        vv.masked_fill_(~past[:, None, :, None], 0.0)
        o = (p @ vv + p_own @ nv) / (p.sum(-1, keepdim=True) + p_own.sum(-1, keepdim=True))
    at = torch.arange(n, device=q.device)
    row = torch.searchsorted(cu[1:], at, right=True)
    o = o.view(rows, hkv, share, top, dh)[row, :, :, at - cu[row]]
    return o.reshape(n, heads, dh).to(q.dtype)


def run(state):
    s = state
    if own:
        return _own(s)
    return {"grow": _plain_grow, "trim": _plain_trim, "append": _plain_append,
            "attend": _plain_attend}[s["kind"]](s)


def _own(s):
    from kernelverify_b200.pack import paged
    if s["kind"] == "grow":
        b = paged.build_tables(s["lens"], s["new"], s["tables"], s["free"], s["n_free"],
                               page_size=s["page"], max_tokens=s["max_tokens"])
        return {"cu_new": b.cu_new, "slots": b.slots, "positions": b.positions, "lens": b.lens,
                "n_free": b.n_free, "status": b.status, "tables": s["tables"]}
    if s["kind"] == "trim":
        lens, n_free = paged.truncate(s["lens"], s["keep"], s["tables"], s["free"], s["n_free"],
                                      page_size=s["page"])
        return {"lens": lens, "n_free": n_free, "free": s["free"]}
    if s["kind"] == "append":
        paged.append(s["new_k"], s["new_v"], *s["k"], *s["v"], s["slots"])
        return list(paged.gather(*s["k"], *s["v"], s["slots"]))
    return paged.attend(s["q"], *s["k"], *s["v"], s["new_k"], s["new_v"], block_tables=s["tables"],
                        ctx_lens=s["ctx"], cu_new=s["cu"], max_new=s["max_new"], max_ctx=s["max_ctx"])


# ---------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(words, scales, biases):
    """Packed rows [rows, W] as float64 [rows, 8 W], one code position at a time."""
    rows, w = words.shape
    group = 8 * w // scales.shape[1]
    wide = words.long() & 0xFFFFFFFF
    out = torch.empty(rows, 8 * w, dtype=torch.float64, device=words.device)
    for i in range(8):
        out[:, i::8] = ((wide >> (4 * i)) % 16).double()
    return out * scales.double().repeat_interleave(group, 1) + biases.double().repeat_interleave(group, 1)


def _exact_append(s):
    """What a quantized row stands for: its codes times its stored scale plus
    its stored bias, the quantizer's steps taken in float32 as its definition
    has them, element by element."""
    out = []
    for pool, x in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        n, hkv, dh = x.shape
        group = dh // pool[1].shape[-1]
        y = x.reshape(-1, group).float().cpu()
        lo, hi = y.min(1).values, y.max(1).values
        hi = torch.maximum(hi, torch.zeros(()))
        width = torch.maximum((hi - lo) / torch.tensor([15.0]), torch.tensor(1e-7))
        neg = lo.abs() > hi.abs()
        edge = torch.where(neg, lo, hi)
        width = torch.where(neg, width, -width)
        ratio = edge / width
        k = torch.trunc(ratio + torch.copysign(torch.full_like(ratio, 0.5), ratio))
        zero = k == 0
        width = torch.where(zero, width, edge / torch.where(zero, torch.ones(()), k))
        edge = torch.where(zero, torch.zeros(()), edge)
        ratio = (y - edge[:, None]) / width[:, None]
        codes = torch.trunc(ratio + torch.copysign(torch.full_like(ratio, 0.5), ratio))
        codes = torch.minimum(codes, torch.tensor(15.0)).double()
        got = codes * width.to(x.dtype).double()[:, None] + edge.to(x.dtype).double()[:, None]
        got = got.reshape(n, hkv, dh)
        got[s["slots"].cpu() < 0] = 0
        out.append(got)
    return out


def _exact_attend(s):
    q, page = s["q"], s["page"]
    n, heads, dh = q.shape
    hkv = s["new_k"].shape[1]
    share = heads // hkv
    out = torch.zeros(n, heads, dh, dtype=torch.float64, device=q.device)
    cu, ctx = s["cu"].tolist(), s["ctx"].tolist()
    for b, length in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        blocks = s["tables"][b, :_pages(length, page)].long()
        causal = torch.ones(hi - lo, hi - lo, device=q.device, dtype=torch.bool).triu(1)
        for h in range(hkv):
            kk, vv = (torch.cat([_exact_values(*[p[blocks, h].reshape(-1, p.shape[-1]) for p in s[x]])[:length],
                                 s["new_" + x][lo:hi, h].double()]) for x in ("k", "v"))
            for j in range(h * share, (h + 1) * share):
                scores = q[lo:hi, j].double() @ kk.T / math.sqrt(dh)
                scores[:, length:].masked_fill_(causal, -math.inf)
                out[lo:hi, j] = torch.softmax(scores, -1) @ vv
    return out


def exact(case, seed):
    if case["kind"] in ("grow", "trim"):
        return None                      # whole numbers only
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(s)
