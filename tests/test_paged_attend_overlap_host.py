"""The paged attention refuses an output or a workspace that lies over one of
its inputs, on a machine without a GPU: its kernels read the lengths, offsets
and tables again while rows and parts are written."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernelverify_b200 import _native

# the addresses are made up: nothing here may get as far as a launch
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="for machines without a GPU")

ROWS, TOKENS, HEADS, KV, DH, GROUP, PAGES, PAGE, WIDTH = 3, 5, 8, 2, 128, 64, 10, 16, 4
RUN = PAGES * KV * PAGE
BYTES = dict(q=TOKENS * HEADS * DH * 2, new_k=TOKENS * KV * DH * 2, new_v=TOKENS * KV * DH * 2,
             k_words=RUN * DH // 2, v_words=RUN * DH // 2, block_tables=4 * ROWS * WIDTH, ctx_lens=4 * ROWS,
             cu_new=4 * ROWS + 4, **{f"{h}_{x}": RUN * (DH // GROUP) * 2 for h in "kv" for x in ("scales", "biases")})
OUT, WS = 1 << 30, 1 << 34


@pytest.fixture(scope="module")
def lib():
    from kernelverify_b200 import build
    build.build()
    return _native.lib()


def args(**over):
    a = _native.KvqPagedArgs()
    for i, name in enumerate(BYTES):
        setattr(a, name, 65536 * (i + 1))
    a.rows, a.tokens, a.n_heads, a.n_kv_heads = ROWS, TOKENS, HEADS, KV
    a.head_dim, a.group_size, a.pages, a.page_size, a.width = DH, GROUP, PAGES, PAGE, WIDTH
    a.max_ctx, a.max_new, a.dtype = WIDTH * PAGE, 3, 0
    a.q_token_stride, a.q_head_stride = HEADS * DH, DH
    a.k_token_stride = a.v_token_stride = KV * DH
    a.k_head_stride = a.v_head_stride = DH
    for k, v in over.items():
        setattr(a, k, v)
    return a


def call(lib, a, out=OUT, ws=WS):
    need = lib.kvq_paged_workspace_bytes(ctypes.byref(a))
    assert need
    return lib.kvq_paged_attend(ctypes.byref(a), out, ws, need, None), need


@pytest.mark.parametrize("name", BYTES)
@pytest.mark.parametrize("what", ["out", "workspace"])
def test_refuses_overlaps(lib, name, what):
    """The input's last bytes on the written range's first, and the reverse."""
    base, (_, need) = (OUT if what == "out" else WS), call(lib, args())
    size = TOKENS * HEADS * DH * 2 if what == "out" else need
    for at in ((base - BYTES[name]) // 16 * 16 + 16, base + size - 16):
        rc, _ = call(lib, args(**{name: at}))
        assert rc == _native.KVQ_ERR_INVALID and b"overlaps" in lib.kvq_last_error()


def test_refuses_a_workspace_over_its_output(lib):
    for ws in (OUT, (OUT + TOKENS * HEADS * DH * 2 - 1) // 256 * 256):
        rc, _ = call(lib, args(), ws=ws)
        assert rc == _native.KVQ_ERR_INVALID and b"overlaps" in lib.kvq_last_error()


@pytest.mark.parametrize("name", BYTES)
def test_neighbours_are_not_refused(lib, name):
    size = -(-BYTES[name] // 16) * 16
    for at in (OUT - size, OUT + TOKENS * HEADS * DH * 2):
        assert call(lib, args(**{name: at}))[0] == _native.KVQ_ERR_UNSUPPORTED
