"""The paged cache's entries on a machine without a GPU: every refusal comes
from the host, before anything could be indexed with a bad argument."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernelverify_b200 import _native
from kernelverify_b200.pack import paged


@pytest.fixture(scope="module")
def lib():
    from kernelverify_b200 import build
    build.build()
    return _native.lib()


def _attend(**over):
    a = _native.KvqPagedArgs()
    for i, name in enumerate(("q", "new_k", "new_v", "k_words", "k_scales", "k_biases", "v_words",
                              "v_scales", "v_biases", "block_tables", "ctx_lens", "cu_new")):
        setattr(a, name, 4096 * (i + 1))
    a.rows, a.tokens, a.n_heads, a.n_kv_heads = 2, 5, 8, 2
    a.head_dim, a.group_size, a.pages, a.page_size, a.width = 128, 64, 10, 16, 4
    a.max_ctx, a.max_new, a.dtype = 64, 3, 0
    a.q_token_stride, a.q_head_stride = 8 * 128, 128
    a.k_token_stride = a.v_token_stride = 2 * 128
    a.k_head_stride = a.v_head_stride = 128
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, needle", [
    (dict(head_dim=96), b"head_dim"), (dict(group_size=48), b"group_size"),
    (dict(head_dim=64, group_size=128), b"divide"), (dict(dtype=2), b"dtype"),
    (dict(page_size=48), b"page_size"), (dict(page_size=256), b"page_size"),
    (dict(pages=0), b"pages"), (dict(n_kv_heads=0), b"cache heads"), (dict(n_heads=7), b"multiple"),
    (dict(rows=0), b"rows"), (dict(rows=4097), b"rows"), (dict(q=None), b"NULL"),
    (dict(cu_new=None), b"NULL"), (dict(v_biases=None), b"NULL"), (dict(k_words=4104), b"16-byte"),
    (dict(q=4097), b"aligned"), (dict(ctx_lens=4098), b"aligned"), (dict(max_ctx=65), b"max_ctx"),
    (dict(tokens=1 << 30), b"too many"),
    (dict(width=1 << 27, max_ctx=0x7FFFFFFE), b"2^31"),
])
def test_attend_refuses(lib, over, needle):
    a = _attend(**over)
    assert lib.kvq_paged_attend(ctypes.byref(a), 8192, None, 0, None) == _native.KVQ_ERR_INVALID
    assert needle in lib.kvq_last_error()
    assert lib.kvq_paged_workspace_bytes(ctypes.byref(a)) == 0


def test_attend_checks_its_output_and_workspace(lib):
    a = _attend()
    assert lib.kvq_paged_attend(ctypes.byref(a), None, None, 0, None) == _native.KVQ_ERR_INVALID
    assert b"out" in lib.kvq_last_error()
    assert lib.kvq_paged_attend(ctypes.byref(a), 8200, None, 0, None) == _native.KVQ_ERR_INVALID
    assert b"16-byte" in lib.kvq_last_error()
    need = lib.kvq_paged_workspace_bytes(ctypes.byref(a))
    if need:
        assert lib.kvq_paged_attend(ctypes.byref(a), 8192, 4096, need - 1, None) == _native.KVQ_ERR_INVALID
        assert b"workspace" in lib.kvq_last_error()
        assert lib.kvq_paged_attend(ctypes.byref(a), 8192, 4112, need, None) == _native.KVQ_ERR_INVALID
        assert b"256-byte" in lib.kvq_last_error()
    assert lib.kvq_paged_attend(None, 8192, None, 0, None) == _native.KVQ_ERR_INVALID


def test_attend_refuses_its_inputs_as_output(lib):
    a = _attend()
    need = lib.kvq_paged_workspace_bytes(ctypes.byref(a))
    for name in ("q", "new_k", "new_v"):
        b = _attend(**{name: (1 << 30) + 256})
        assert lib.kvq_paged_attend(ctypes.byref(b), 1 << 30, 1 << 20, need, None) == _native.KVQ_ERR_INVALID
        assert b"overlaps" in lib.kvq_last_error()


def _tables(**over):
    t = _native.KvqTables()
    for i, (name, _) in enumerate(_native.KvqTables._fields_[:11]):
        setattr(t, name, 65536 * (i + 1))
    t.rows, t.width, t.pool, t.page_size, t.max_tokens = 8, 4, 100, 16, 50
    for k, v in over.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("over, needle", [
    (dict(lens=None), b"NULL"), (dict(slots=None), b"NULL"), (dict(status=None), b"NULL"),
    (dict(page_size=8), b"page_size"), (dict(rows=0), b"rows"), (dict(rows=4097), b"rows"),
    (dict(pool=0), b"stack"), (dict(width=0), b"columns"), (dict(width=1 << 28), b"columns"),
    (dict(rows=4096, width=1 << 20), b"columns"), (dict(lens=65538), b"aligned"),
    (dict(slots=65540), b"aligned"), (dict(lens_out=65536), b"overlaps"),
    (dict(lens_out=65536 + 4), b"overlaps"), (dict(n_free_out=65536 * 5), b"overlaps"),
    (dict(cu_new=65536 * 2 - 32), b"overlaps"), (dict(max_tokens=1 << 31), b"max_tokens"),
])
def test_tables_refuse(lib, over, needle):
    t = _tables(**over)
    assert lib.kvq_paged_tables(ctypes.byref(t), None) == _native.KVQ_ERR_INVALID
    assert needle in lib.kvq_last_error()


@pytest.mark.parametrize("over, needle", [
    (dict(step=None), b"NULL"), (dict(lens_out=65536 * 2), b"overlaps"), (dict(page_size=0), b"page_size"),
])
def test_truncate_refuses(lib, over, needle):
    t = _tables(**over)
    assert lib.kvq_paged_truncate(ctypes.byref(t), None) == _native.KVQ_ERR_INVALID
    assert needle in lib.kvq_last_error()


def _rows(**over):
    r = _native.KvqPagedRows()
    for i, (name, _) in enumerate(_native.KvqPagedRows._fields_[:9]):
        setattr(r, name, 4096 * (i + 1))
    r.tokens, r.n_kv_heads, r.head_dim, r.group_size = 5, 2, 128, 64
    r.pages, r.page_size, r.dtype, r.out_dtype = 10, 16, 0, 0
    for k, v in over.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("over, needle", [
    (dict(head_dim=32), b"head_dim"), (dict(page_size=24), b"page_size"), (dict(slots=None), b"NULL"),
    (dict(keys=None), b"NULL"), (dict(k_scales=4100), b"16-byte"), (dict(slots=4100), b"aligned"),
    (dict(tokens=1 << 31), b"tokens"), (dict(dtype=7), b"dtype"),
])
def test_rows_refuse(lib, over, needle):
    for entry in (lib.kvq_paged_append, lib.kvq_paged_gather):
        assert entry(ctypes.byref(_rows(**over)), None) == _native.KVQ_ERR_INVALID
        assert needle in lib.kvq_last_error()


def test_rows_refuse_by_direction(lib):
    assert lib.kvq_paged_append(ctypes.byref(_rows(keys=4097)), None) == _native.KVQ_ERR_INVALID
    assert lib.kvq_paged_gather(ctypes.byref(_rows(keys=4104)), None) == _native.KVQ_ERR_INVALID
    assert lib.kvq_paged_gather(ctypes.byref(_rows(dtype=1, out_dtype=0)), None) == _native.KVQ_ERR_INVALID
    assert b"out_dtype" in lib.kvq_last_error()


def test_no_device_is_a_status(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for entry, a in ((lib.kvq_paged_tables, _tables()), (lib.kvq_paged_truncate, _tables()),
                     (lib.kvq_paged_append, _rows()), (lib.kvq_paged_gather, _rows())):
        assert entry(ctypes.byref(a), None) == _native.KVQ_ERR_UNSUPPORTED
    a = _attend()
    need = lib.kvq_paged_workspace_bytes(ctypes.byref(a))
    assert lib.kvq_paged_attend(ctypes.byref(a), 1 << 30, 1 << 20, need, None) == _native.KVQ_ERR_UNSUPPORTED


def test_python_refuses_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.build_tables(i, i, torch.zeros(2, 3, dtype=torch.int32), i, i[:1], page_size=16, max_tokens=4)
    with pytest.raises(ValueError, match="CUDA"):
        paged.truncate(i, i, torch.zeros(2, 3, dtype=torch.int32), i, i[:1], page_size=16)
    w = torch.zeros(1, 1, 16, 16, dtype=torch.int32)
    s = torch.zeros(1, 1, 16, 2, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.gather(w, s, s, w, s, s, torch.zeros(1, dtype=torch.int64))


def test_serving_classes_check_their_arguments():
    from kernelverify_b200 import serving
    seqs = serving.PagedSequences(3, 10, 100, 16, device="cpu")
    assert seqs.width == 7 and seqs.n_free.item() == 10 and seqs.block_tables.shape == (3, 7)
    cache = serving.PagedKVCache(seqs, 2, 64, 32)
    assert cache.keys[0].shape == (10, 2, 16, 8) and cache.values[1].shape == (10, 2, 16, 2)
    assert cache.nbytes() == 10 * 2 * 16 * 2 * (32 + 2 * 2 * 2)
    for bad in (dict(batch=0), dict(pages=0), dict(max_len=0), dict(page_size=20), dict(batch=5000)):
        with pytest.raises(ValueError):
            serving.PagedSequences(**(dict(batch=3, pages=10, max_len=100, device="cpu") | bad))
    for bad in (dict(head_dim=96), dict(head_dim=64, group_size=128)):
        with pytest.raises(ValueError):
            serving.PagedKVCache(seqs, **(dict(n_kv_heads=2, head_dim=64) | bad))


def test_packed_argument_blocks_are_the_structures():
    """The blocks that are packed by hand have the C structures' layout."""
    for form, struct_type in ((paged._TABLES, _native.KvqTables), (paged._ROWS, _native.KvqPagedRows),
                              (paged._ARGS, _native.KvqPagedArgs)):
        assert form.size == ctypes.sizeof(struct_type)
        names = [n for n, _ in struct_type._fields_]
        got = struct_type.from_buffer_copy(form.pack(*range(1, len(names) + 1)))
        assert [getattr(got, n) for n in names] == list(range(1, len(names) + 1))
