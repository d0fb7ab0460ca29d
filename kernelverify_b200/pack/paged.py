"""Paged 4-bit K/V cache: block tables, append, read-back and attention.

The packed rows of `kv_attention` (MLX-affine 4-bit codes with a scale and a
bias per group), held in pages that the requests of a batch take and give
back, over the C ABI's `kvq_paged_*` entries. A serving step is

    batch = build_tables(lens, new_lens, block_tables, free_pages, n_free, ...)
    append(keys, values, *k_pool, *v_pool, batch.slots)
    out = attend(q, *k_pool, *v_pool, keys, values, block_tables=block_tables,
                 ctx_lens=lens, cu_new=batch.cu_new, max_new=...)

per layer for the last two, and `truncate` gives pages back: a finished
request's, or a rejected draft's. None of it needs the host to know the
lengths, so a step can be captured as a CUDA graph.

A pool half is a triplet (words int32 [pages, HKV, page_size, DH/8], scales
and biases [pages, HKV, page_size, DH/group]) in float16 or float32; slot s is
position s % page_size of page s // page_size.

No reference counterpart: its cache is one padded buffer per sequence
(kernelverify/pack/kv_attention.py:85-234 reads it whole).
"""

from __future__ import annotations

import struct
from typing import NamedTuple

from kernelverify_b200 import _native
from kernelverify_b200.pack.kv_attention import (SUPPORTED_DH, SUPPORTED_GROUPS, Workspace,
                                                 _dtype_code)

BITS = 4
PAGE_SIZES = (16, 32, 64, 128)
MAX_ROWS = 4096
# bits of PageBatch.status
POOL_EMPTY, ROW_FULL, TOO_MANY_TOKENS = 1, 2, 4

# The C argument blocks (kvq_tables, kvq_paged_rows, kvq_paged_args), packed in
# one go: a step makes two of these calls per layer, and the host's part of a
# call is most of a small step's time.
_TABLES = struct.Struct("@11Q5I4x")
_ROWS = struct.Struct("@13Q8I")
_ARGS = struct.Struct("@18Q12I")

_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


class PageBatch(NamedTuple):
    """A step's tables, all on the device: `cu_new` int32 [B + 1] running sums
    of the new tokens, `slots` int64 and `positions` int32 [max_tokens] per
    token (-1 and 0 past the last one), `lens` int32 [B] and `n_free` int32 [1]
    after the step, `status` int32 [1]: 0, or the POOL_EMPTY / ROW_FULL /
    TOO_MANY_TOKENS bits of a step that did not fit and took nothing."""
    cu_new: object
    slots: object
    positions: object
    lens: object
    n_free: object
    status: object


def _check(name, ten, shape, dtype, device) -> None:
    """A contiguous tensor of exactly this shape and dtype on CUDA device
    `device` (its index; the library indexes it by its address alone)."""
    if ten.shape != shape:
        raise ValueError(f"{name} has shape {tuple(ten.shape)}, expected {tuple(shape)}")
    if ten.dtype != dtype:
        raise ValueError(f"{name} is {ten.dtype}, expected {dtype}")
    if not ten.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if ten.get_device() != device:
        raise ValueError(f"{name} is on {ten.device}, expected cuda:{device}")


def _cuda_device(name, ten) -> int:
    device = ten.get_device()
    if device < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return device


def _page_size(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} not in {PAGE_SIZES}")
    return page_size


def _call(entry, device, stream, *args) -> None:
    """entry(*args, stream handle) with `device` current, so a tensor's device
    decides where the kernel runs, not the caller's current one."""
    torch = _torch()
    if torch._C._cuda_getDevice() == device:
        _native.check(entry(*args, stream.cuda_stream if stream is not None
                            else torch._C._cuda_getCurrentRawStream(device)))
        return
    with torch.cuda.device(device):
        _native.check(entry(*args, stream.cuda_stream if stream is not None
                            else torch._C._cuda_getCurrentRawStream(device)))


def _empty(stream, like, shape, dtype):
    """An unwritten tensor on `like`'s device whose memory belongs to `stream`
    (None: the current one), so that it is reused after that stream's work."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _tables(lens, step, block_tables, free_pages, n_free, page_size):
    """Checked common arguments of build_tables / truncate: (device, rows, values)."""
    i32 = _torch().int32
    device = _cuda_device("lens", lens)
    if lens.dim() != 1:
        raise ValueError(f"lens must be [B], got {tuple(lens.shape)}")
    rows = lens.shape[0]
    if not 1 <= rows <= MAX_ROWS:
        raise ValueError(f"{rows} requests: 1 to {MAX_ROWS}")
    if block_tables.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_tables must be [B, W] and free_pages [pages]")
    width, pool = block_tables.shape[1], free_pages.shape[0]
    if not (step.shape == (rows,) and n_free.shape == (1,) and block_tables.shape[0] == rows
            and lens.dtype == step.dtype == block_tables.dtype == free_pages.dtype == n_free.dtype == i32
            and lens.is_contiguous() and step.is_contiguous() and block_tables.is_contiguous()
            and free_pages.is_contiguous()
            and step.get_device() == block_tables.get_device() == free_pages.get_device()
            == n_free.get_device() == device):
        # something is off: find out what
        _check("lens", lens, (rows,), i32, device)
        _check("block_tables", block_tables, (rows, width), i32, device)
        _check("free_pages", free_pages, (pool,), i32, device)
        _check("n_free", n_free, (1,), i32, device)
        _check("new_lens or keep", step, (rows,), i32, device)
    _page_size(page_size)
    return device, rows, width, pool


def _batch(stream, like, rows: int, max_tokens: int) -> PageBatch:
    torch = _torch()
    cu, lens, n_free, status, pos = _empty(
        stream, like, 2 * rows + 3 + max_tokens, torch.int32).split_with_sizes(
            [rows + 1, rows, 1, 1, max_tokens])
    return PageBatch(cu, _empty(stream, like, max_tokens, torch.int64), pos, lens, n_free, status)


def empty_batch(rows: int, max_tokens: int, device) -> PageBatch:
    """Unwritten buffers of a step's tables, for `build_tables(out=...)`."""
    return _batch(None, _torch().empty(0, device=device), rows, max_tokens)


def build_tables(lens, new_lens, block_tables, free_pages, n_free, *, page_size: int,
                 max_tokens: int, out: PageBatch | None = None, stream=None) -> PageBatch:
    """Tables, slots and positions of a step in which request b, holding
    lens[b] positions, brings new_lens[b] tokens (int32 [B], on the device;
    negative counts as 0).

    The pages that are lacking come from the top of the stack
    free_pages[0 .. n_free) (int32 [pages], int32 [1]), requests in order, and
    are written into `block_tables` (int32 [B, W]) in place; `lens` and
    `n_free` are not changed, the returned batch has them as they are after the
    step. A step that does not fit takes nothing and says so in `status`, which
    the caller reads when it suits it: its slots are -1 and its `cu_new` 0, so
    the step's `append` and `attend` do nothing."""
    device, rows, width, pool = _tables(lens, new_lens, block_tables, free_pages, n_free, page_size)
    if not 0 <= max_tokens < 2 ** 31:
        raise ValueError(f"max_tokens {max_tokens} is outside [0, 2^31)")
    if out is None:
        out = _batch(stream, lens, rows, max_tokens)
    else:
        torch = _torch()
        _check("out.slots", out.slots, (max_tokens,), torch.int64, device)
        for name, n in (("cu_new", rows + 1), ("positions", max_tokens), ("lens", rows),
                        ("n_free", 1), ("status", 1)):
            _check("out." + name, getattr(out, name), (n,), torch.int32, device)
    _call(_native.lib().kvq_paged_tables, device, stream, _TABLES.pack(
        lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
        n_free.data_ptr(), out.cu_new.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(),
        out.lens.data_ptr(), out.n_free.data_ptr(), out.status.data_ptr(), rows, width, pool,
        page_size, max_tokens))
    return out


def truncate(lens, keep, block_tables, free_pages, n_free, *, page_size: int, out=None,
             stream=None):
    """Cut request b to min(lens[b], keep[b]) positions (int32 [B]; negative
    counts as 0: all of it goes) and push the pages behind them on the stack
    free_pages[n_free ..], in place. Returns (lens int32 [B], n_free int32 [1])
    after it, or fills `out` of the same form; `lens` and `n_free` are not
    changed, nor are the tables' entries."""
    device, rows, width, pool = _tables(lens, keep, block_tables, free_pages, n_free, page_size)
    torch = _torch()
    if out is None:
        lens_out, n_out = _empty(stream, lens, rows + 1, torch.int32).split_with_sizes([rows, 1])
    else:
        lens_out, n_out = out
        _check("out[0]", lens_out, (rows,), torch.int32, device)
        _check("out[1]", n_out, (1,), torch.int32, device)
    _call(_native.lib().kvq_paged_truncate, device, stream, _TABLES.pack(
        lens.data_ptr(), keep.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
        n_free.data_ptr(), 0, 0, 0, lens_out.data_ptr(), n_out.data_ptr(), 0, rows, width, pool,
        page_size, 0))
    return lens_out, n_out


def _pools(k_wq, k_scales, k_biases, v_wq, v_scales, v_biases):
    """Checked pools: (device, dtype, pages, heads, page size, head dim, group,
    the six addresses)."""
    torch = _torch()
    device = _cuda_device("k_wq", k_wq)
    if k_wq.dim() != 4 or k_scales.dim() != 4:
        raise ValueError(f"a pool's tensors must be [pages, HKV, page_size, ...], got "
                         f"{tuple(k_wq.shape)} and {tuple(k_scales.shape)}")
    pages, heads, page, words = k_wq.shape
    head_dim, groups = words * 8, k_scales.shape[3]
    if head_dim not in SUPPORTED_DH:
        raise ValueError(f"head_dim {head_dim} (8 codes of {BITS} bits per word) not in {SUPPORTED_DH}")
    if page not in PAGE_SIZES:
        raise ValueError(f"page_size {page} not in {PAGE_SIZES}")
    if groups == 0 or head_dim % groups or head_dim // groups not in SUPPORTED_GROUPS:
        raise ValueError(f"{groups} groups per row: group_size must be one of {SUPPORTED_GROUPS}")
    dtype, wdt, shape, lead = k_scales.dtype, k_wq.dtype, k_wq.shape, k_scales.shape
    if wdt != torch.int32 and wdt != torch.uint32:
        raise ValueError("packed words must be int32/uint32 tensors")
    if lead[:3] != shape[:3]:
        raise ValueError(f"k_scales has shape {tuple(lead)}, expected {tuple(shape[:3])} first")
    if not (v_wq.shape == shape and k_biases.shape == v_scales.shape == v_biases.shape == lead
            and v_wq.dtype == wdt and k_biases.dtype == v_scales.dtype == v_biases.dtype == dtype
            and k_wq.is_contiguous() and v_wq.is_contiguous() and k_scales.is_contiguous()
            and k_biases.is_contiguous() and v_scales.is_contiguous() and v_biases.is_contiguous()
            and v_wq.get_device() == k_scales.get_device() == k_biases.get_device()
            == v_scales.get_device() == v_biases.get_device() == device):
        # something is off: find out what
        for name, ten, want, kind in (("k_wq", k_wq, shape, wdt), ("v_wq", v_wq, shape, wdt),
                                      ("k_scales", k_scales, lead, dtype),
                                      ("k_biases", k_biases, lead, dtype),
                                      ("v_scales", v_scales, lead, dtype),
                                      ("v_biases", v_biases, lead, dtype)):
            _check(name, ten, want, kind, device)
    return (device, dtype, pages, heads, page, head_dim, head_dim // groups,
            (k_wq.data_ptr(), k_scales.data_ptr(), k_biases.data_ptr(), v_wq.data_ptr(),
             v_scales.data_ptr(), v_biases.data_ptr()))


def _rows(name, ten, shape, dtype, device):
    """Checked [tokens, heads, DH] rows with DH contiguous, any token and head
    stride: (address, token stride, head stride)."""
    if ten.shape != shape:
        raise ValueError(f"{name} has shape {tuple(ten.shape)}, expected {tuple(shape)}")
    if ten.dtype != dtype:
        raise ValueError(f"{name} is {ten.dtype}; the cache holds {dtype}")
    if ten.get_device() != device:
        raise ValueError(f"{name} is on {ten.device}, expected cuda:{device}")
    token, head, dim = ten.stride()
    if dim != 1:
        raise ValueError(f"{name}'s head_dim must be contiguous")
    if token < 0 or head < 0:
        raise ValueError(f"{name} has a negative stride")
    return ten.data_ptr(), token, head


def append(keys, values, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, slots, *,
           stream=None) -> None:
    """Quantize keys / values [N, HKV, DH] into their slots (int64 [N]) of the
    pools, in place; bit for bit the rows `kv_attention.quantize_cache` makes.
    A slot below 0 or past the pool is skipped (a padded step's tokens). Two
    tokens must not name the same slot."""
    device, dtype, pages, heads, page, head_dim, group, pool = _pools(
        k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    if keys.dim() != 3:
        raise ValueError(f"keys must be [N, HKV, DH], got {tuple(keys.shape)}")
    n = keys.shape[0]
    kp, kt, kh = _rows("keys", keys, (n, heads, head_dim), dtype, device)
    vp, vt, vh = _rows("values", values, (n, heads, head_dim), dtype, device)
    _check("slots", slots, (n,), _torch().int64, device)
    code = _dtype_code(dtype)
    _call(_native.lib().kvq_paged_append, device, stream, _ROWS.pack(
        *pool, kp, vp, slots.data_ptr(), kt, kh, vt, vh, n, heads, head_dim, group, pages, page,
        code, code))


def gather(k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, slots, *, dtype=None, stream=None):
    """(keys, values) [N, HKV, DH] that the slots (int64 [N]) hold, dequantized
    (scale * code + bias in float32) into `dtype`: the cache's (the default) or
    float32. A slot below 0 or past the pool reads as zeros."""
    torch = _torch()
    device, held, pages, heads, page, head_dim, group, pool = _pools(
        k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    if slots.dim() != 1:
        raise ValueError(f"slots must be [N], got {tuple(slots.shape)}")
    n = slots.shape[0]
    _check("slots", slots, (n,), torch.int64, device)
    dtype = held if dtype is None else dtype
    if dtype != held and dtype != torch.float32:
        raise ValueError(f"dtype {dtype}: the cache's {held} or float32")
    out = _empty(stream, k_wq, (2, n, heads, head_dim), dtype)
    keys, values = out.unbind(0)
    _call(_native.lib().kvq_paged_gather, device, stream, _ROWS.pack(
        *pool, keys.data_ptr(), values.data_ptr(), slots.data_ptr(), 0, 0, 0, 0, n, heads,
        head_dim, group, pages, page, _dtype_code(held), _dtype_code(dtype)))
    return keys, values


def attend(q, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, new_k, new_v, *, block_tables,
           ctx_lens, cu_new, max_new: int, max_ctx: int | None = None, out=None,
           workspace: Workspace | None = None, stream=None):
    """The step's attention: out [N, H, DH] in q's dtype.

    Request b brings the tokens cu_new[b] .. cu_new[b+1) (int32 [B + 1]) of
    q [N, H, DH] and new_k / new_v [N, HKV, DH] (head_dim contiguous, any other
    strides); its i-th token sees the ctx_lens[b] positions (int32 [B]) that
    the cache held before the step, through block_tables (int32 [B, W]), and
    the step's own entries 0..i of the request at full precision -- with one
    token, the step of `kv_attention.decode`. Scores are scaled by
    1/sqrt(DH); query head h reads cache head h // (H // HKV).

    `max_new` bounds a request's new tokens and `max_ctx` (default: W pages)
    its cached positions; the launch is sized by them and longer requests are
    cut to them. Rows of `out` past the last request's tokens are not written;
    an `out` that overlaps an input is refused.
    A page id outside the pool makes the rows that need it NaN. An own entry that
    is not finite reaches the tokens that see it alone: a key's infinity as a score
    of +inf (a row that is not finite) or -inf (as without the entry). Float32
    inputs are of magnitudes below 2^60."""
    torch = _torch()
    device, dtype, pages, heads, page, head_dim, group, pool = _pools(
        k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    if q.dim() != 3:
        raise ValueError(f"q must be [N, H, DH], got {tuple(q.shape)}")
    n, n_heads = q.shape[0], q.shape[1]
    if n_heads == 0 or n_heads % heads:
        raise ValueError(f"{n_heads} query heads do not divide into {heads} cache heads")
    qp, qt, qh = _rows("q", q, (n, n_heads, head_dim), dtype, device)
    kp, kt, kh = _rows("new_k", new_k, (n, heads, head_dim), dtype, device)
    vp, vt, vh = _rows("new_v", new_v, (n, heads, head_dim), dtype, device)
    i32 = torch.int32
    if block_tables.dim() != 2:
        raise ValueError(f"block_tables must be [B, W], got {tuple(block_tables.shape)}")
    rows, width = block_tables.shape
    if not 1 <= rows <= MAX_ROWS:
        raise ValueError(f"{rows} requests: 1 to {MAX_ROWS}")
    if not (ctx_lens.shape == (rows,) and cu_new.shape == (rows + 1,)
            and block_tables.dtype == ctx_lens.dtype == cu_new.dtype == i32
            and block_tables.is_contiguous() and ctx_lens.is_contiguous() and cu_new.is_contiguous()
            and block_tables.get_device() == ctx_lens.get_device() == cu_new.get_device() == device):
        # something is off: find out what
        _check("block_tables", block_tables, block_tables.shape, i32, device)
        _check("ctx_lens", ctx_lens, (rows,), i32, device)
        _check("cu_new", cu_new, (rows + 1,), i32, device)
    if max_ctx is None:
        max_ctx = width * page
    if not 0 <= max_ctx <= width * page:
        raise ValueError(f"max_ctx {max_ctx} is outside [0, {width * page}]: the tables hold {width} pages")
    if not 0 <= max_new < 2 ** 31:
        raise ValueError(f"max_new {max_new} is outside [0, 2^31)")
    if out is None:
        out = _empty(stream, q, (n, n_heads, head_dim), dtype)
    else:
        _check("out", out, (n, n_heads, head_dim), dtype, device)
    a = _ARGS.pack(qp, kp, vp, *pool, block_tables.data_ptr(), ctx_lens.data_ptr(),
                   cu_new.data_ptr(), qt, qh, kt, kh, vt, vh, rows, n, n_heads, heads, head_dim,
                   group, pages, page, width, max_ctx, max_new, _dtype_code(dtype))
    lib = _native.lib()
    need = lib.kvq_paged_workspace_bytes(a)
    ws, have = None, 0
    if need:
        # a buffer of the call's own unless the caller keeps one: the allocator
        # orders its reuse after this call, and a captured step's is its graph's
        if workspace is None:
            buf, have = _empty(stream, q, need, torch.uint8), need
        else:
            buf, have = workspace.get(need, q.device, stream)
        ws = buf.data_ptr()
    _call(lib.kvq_paged_attend, device, stream, a, out.data_ptr(), ws, have)
    return out
