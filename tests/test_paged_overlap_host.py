"""Block tables and truncate refuse tensors that lie over one another, on a
machine without a GPU: every CTA reads the inputs while others write."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernelverify_b200 import _native

# the addresses are made up: nothing here may get as far as a launch
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="for machines without a GPU")


@pytest.fixture(scope="module")
def lib():
    from kernelverify_b200 import build
    build.build()
    return _native.lib()


NAMES = [name for name, _ in _native.KvqTables._fields_[:11]]
ROWS, WIDTH, POOL, TOKENS = 8, 4, 100, 50
BYTES = dict(lens=4 * ROWS, step=4 * ROWS, block_tables=4 * ROWS * WIDTH, free_pages=4 * POOL, n_free=4,
             cu_new=4 * ROWS + 4, slots=8 * TOKENS, positions=4 * TOKENS, lens_out=4 * ROWS, n_free_out=4, status=4)
BUILD_WRITES = ("block_tables", "cu_new", "slots", "positions", "lens_out", "n_free_out", "status")
TRUNCATE_WRITES = ("free_pages", "lens_out", "n_free_out")
TRUNCATE_USES = ("lens", "step", "block_tables", "free_pages", "n_free", "lens_out", "n_free_out")


def tables(**over):
    t = _native.KvqTables()
    for i, name in enumerate(NAMES):
        setattr(t, name, 65536 * (i + 1))
    t.rows, t.width, t.pool, t.page_size, t.max_tokens = ROWS, WIDTH, POOL, 16, TOKENS
    for k, v in over.items():
        setattr(t, k, v)
    return t


def refused(entry, lib, t):
    return entry(ctypes.byref(t), None) == _native.KVQ_ERR_INVALID and b"overlap" in lib.kvq_last_error()


def pairs(writes, uses):
    return [(w, u) for w in writes for u in uses if u != w]


@pytest.mark.parametrize("written, other", pairs(BUILD_WRITES, NAMES))
def test_build_tables_refuses_overlaps(lib, written, other):
    """The written tensor's last byte on the other's first, and the reverse."""
    at = getattr(tables(), other)
    unit = 8 if written == "slots" else 4
    assert refused(lib.kvq_paged_tables, lib, tables(**{written: at - BYTES[written] + unit}))
    last = at + BYTES[other] - 4
    assert refused(lib.kvq_paged_tables, lib, tables(**{written: last // unit * unit}))


@pytest.mark.parametrize("written, other", pairs(TRUNCATE_WRITES, TRUNCATE_USES))
def test_truncate_refuses_overlaps(lib, written, other):
    at = getattr(tables(), other)
    assert refused(lib.kvq_paged_truncate, lib, tables(**{written: at - BYTES[written] + 4}))
    assert refused(lib.kvq_paged_truncate, lib, tables(**{written: at + BYTES[other] - 4}))


@pytest.mark.parametrize("entry, uses", [("kvq_paged_tables", NAMES), ("kvq_paged_truncate", TRUNCATE_USES)])
def test_neighbours_are_not_refused(lib, entry, uses):
    """Tensors that lie side by side in one buffer pass every check (and find no
    device); what is not an argument of the entry may lie anywhere."""
    at, top = {}, 1 << 20
    for name in ("slots", *(n for n in NAMES if n != "slots")):
        at[name] = top if name in uses else 1 << 20
        top += BYTES[name] if name in uses else 0
    assert getattr(lib, entry)(ctypes.byref(tables(**at)), None) == _native.KVQ_ERR_UNSUPPORTED
