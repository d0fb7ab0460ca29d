"""The paged cache's five operators in plain form on CPU tensors, so that the
host's part of the serving classes runs on a machine without a GPU."""

from __future__ import annotations

import math

import numpy as np
import torch

from kernelverify_b200.pack import paged
from oracle import quant
from tests import paged_cases as pc


def _put(dst, values):
    dst.copy_(torch.tensor(values, dtype=dst.dtype).view(dst.shape))


def build_tables(lens, new_lens, block_tables, free_pages, n_free, *, page_size, max_tokens, out=None, stream=None):
    rows = lens.numel()
    if out is None:
        i32 = torch.int32
        out = paged.PageBatch(*(torch.empty(n, dtype=t) for n, t in (
            (rows + 1, i32), (max_tokens, torch.int64), (max_tokens, i32), (rows, i32), (1, i32), (1, i32))))
    *parts, tables = pc.tables_reference(lens.tolist(), new_lens.tolist(), block_tables.tolist(),
                                         free_pages.tolist(), int(n_free), page_size, max_tokens)
    for dst, values in zip(out, parts):
        _put(dst, values)
    _put(block_tables, tables)
    return out


def truncate(lens, keep, block_tables, free_pages, n_free, *, page_size, out=None, stream=None):
    got, height, stack = pc.truncate_reference(lens.tolist(), keep.tolist(), block_tables.tolist(),
                                               free_pages.tolist(), int(n_free), page_size)
    _put(free_pages, stack)
    return torch.tensor(got, dtype=torch.int32), torch.tensor([height], dtype=torch.int32)


def append(keys, values, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, slots, *, stream=None):
    page = k_wq.shape[2]
    for x, pool in ((keys, (k_wq, k_scales, k_biases)), (values, (v_wq, v_scales, v_biases))):
        n, heads, dh = x.shape
        if n == 0:
            continue
        codes, s, z = quant.canonical_quantize(x.reshape(-1, dh).numpy(), 4, dh // pool[1].shape[3])
        rows = (quant.pack_codes(codes, 4).view(np.int32), s, z)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < k_wq.shape[0] * page:
                for dst, r in zip(pool, rows):
                    dst[slot // page, :, slot % page] = torch.from_numpy(r[i * heads:(i + 1) * heads])


def gather(k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, slots, *, dtype=None, stream=None):
    page, heads, dh = k_wq.shape[2], k_wq.shape[1], k_wq.shape[3] * 8
    out = []
    for w, s, z in ((k_wq, k_scales, k_biases), (v_wq, v_scales, v_biases)):
        live = (slots >= 0) & (slots < w.shape[0] * page)
        at = slots.clamp(0, w.shape[0] * page - 1)
        rows = [x[at // page, :, at % page].reshape(-1, x.shape[3]).numpy() for x in (w, s, z)]
        codes = quant.unpack_codes(rows[0].view(np.uint32), 4, dh)
        x = torch.from_numpy(quant.dequantize(codes, rows[1], rows[2], dh // s.shape[3], np.float32))
        out.append((x.view(-1, heads, dh) * live[:, None, None]).to(dtype or s.dtype))
    return tuple(out)


def attend(q, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, new_k, new_v, *, block_tables, ctx_lens, cu_new,
           max_new, max_ctx=None, out=None, workspace=None, stream=None):
    page, share = k_wq.shape[2], q.shape[1] // k_wq.shape[1]
    out = torch.full_like(q, 7.0) if out is None else out
    cu = cu_new.tolist()
    for b, length in enumerate(ctx_lens.tolist()):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        pos = torch.arange(length)
        k, v = gather(k_wq, k_scales, k_biases, v_wq, v_scales, v_biases,
                      block_tables[b, pos // page].long() * page + pos % page, dtype=torch.float32)
        k, v = (torch.cat([x, y[lo:hi].float()]).repeat_interleave(share, 1) for x, y in ((k, new_k), (v, new_v)))
        s = torch.einsum("ihd,jhd->hij", q[lo:hi].float(), k) / math.sqrt(q.shape[2])
        s[:, :, length:].masked_fill_(torch.ones(hi - lo, hi - lo, dtype=torch.bool).triu(1), -math.inf)
        out[lo:hi] = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).to(q.dtype)
    return out


def install(monkeypatch) -> None:
    for fn in (build_tables, truncate, append, gather, attend):
        monkeypatch.setattr(paged, fn.__name__, fn)
