"""The paged cache's operators on the device against plain implementations in
64 bits (or whole numbers): sizes and lengths where they can go wrong, padding,
strides, streams, captured steps, and a serving step of all of them."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from kernelverify_b200.pack import kv_attention as kva
from kernelverify_b200.pack import paged
from oracle import quant
from tests import paged_cases as pc
from tests.paged_cases import Step, cdiv

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _needs(native):
    torch.manual_seed(0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _held(rng, lens, page, width, spare):
    """Random tables for `lens` and the stack of the pages left."""
    need = [cdiv(max(n, 0), page) for n in lens]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return tables, order[at:] + [-1] * sum(need), len(order) - at


TABLE_CASES = [
    # lens, new, page, padding
    ([0], [1], 16, 0), ([0], [0], 16, 3), ([15], [1], 16, 0), ([16], [1], 16, 0), ([17], [64], 32, 5),
    ([0, 0, 0, 5], [0, 3, 0, 0], 16, 1), ([31, 64, 0, 63, 1], [1, 1, 1, 1, 1], 64, 0),
    ([5, -3, 7], [-2, 4, 130], 128, 2), (list(range(33)), list(range(33, 0, -1)), 16, 0),
    ([0] * 700, [1, 0, 17, 40, 2] * 140, 16, 77), ([100] * 4096, [1] * 4096, 64, 0),
    ([9000, 0], [1, 20000], 16, 0),
]


@pytest.mark.parametrize("lens, new, page, pad", TABLE_CASES)
def test_build_tables(lens, new, page, pad):
    rng = random.Random(len(lens) + page)
    width = max(1, max(cdiv(max(a, 0) + max(n, 0), page) for a, n in zip(lens, new)))
    lack = sum(cdiv(max(a, 0) + max(n, 0), page) - cdiv(max(a, 0), page) for a, n in zip(lens, new))
    tables, free, n_free = _held(rng, lens, page, width, lack + rng.randint(0, 3) or 1)
    tokens = sum(max(n, 0) for n in new) + pad
    t, f, lt, nt = i32(tables), i32(free), i32(lens), i32(new)
    for _ in range(2):                       # a second call finds what the first one left
        got = paged.build_tables(lt, nt, t, f, i32([n_free]), page_size=page, max_tokens=tokens)
        want = pc.tables_reference(lens, new, tables, free, n_free, page, tokens)
        for name, x, w in zip(("cu_new", "slots", "positions", "lens", "n_free", "status"), got, want):
            assert x.flatten().tolist() == (w if isinstance(w, list) else [w]), name
        assert t.tolist() == want[-1]
    assert lt.tolist() == lens and f.tolist() == free


@pytest.mark.parametrize("lens, new, width, spare, tokens, status", [
    ([16, 3], [17, 1], 4, 1, 40, 1), ([16, 3], [50, 1], 4, 9, 60, 2), ([16, 3], [17, 1], 4, 9, 17, 4),
    ([16, 3], [500, 1], 4, 1, 17, 7), ([2 ** 31 - 1, 0], [2 ** 31 - 1, 1], 4, 1, 5, 7),
])
def test_build_tables_that_do_not_fit_take_nothing(lens, new, width, spare, tokens, status):
    tables = [[1, 2, -1, -1], [3, -1, -1, -1]]
    t, f = i32(tables), i32([9] * spare)
    got = paged.build_tables(i32(lens), i32(new), t, f, i32([spare]), page_size=16, max_tokens=tokens)
    assert got.status.item() == status
    assert got.cu_new.tolist() == [0, 0, 0] and set(got.slots.tolist()) == {-1}
    assert got.lens.tolist() == lens and got.n_free.item() == spare and t.tolist() == tables


@pytest.mark.parametrize("lens, keep, page", [
    ([0], [0], 16), ([1], [0], 16), ([16, 17, 33], [15, 16, 17], 16), ([100, 5, 0, 64], [100, 9, 3, -4], 32),
    ([8192] * 300, [0] * 300, 16), (list(range(0, 4096)), [7] * 4096, 64), ([70000, 2], [3, 0], 16),
])
def test_truncate(lens, keep, page):
    rng = random.Random(3)
    width = max(1, max(cdiv(n, page) for n in lens))
    tables, free, n_free = _held(rng, lens, page, width, 2)
    t, f, lt = i32(tables), i32(free), i32(lens)
    got_lens, got_free = paged.truncate(lt, i32(keep), t, f, i32([n_free]), page_size=page)
    want = pc.truncate_reference(lens, keep, tables, free, n_free, page)
    assert got_lens.tolist() == want[0] and got_free.item() == want[1] and f.tolist() == want[2]
    assert t.tolist() == tables and lt.tolist() == lens


def test_tables_reuse_buffers_and_refuse_their_inputs():
    lens, n_free = i32([5, 0]), i32([4])
    t, f = i32([[0, -1], [-1, -1]]), i32([3, 4, 5, 6])
    out = paged.empty_batch(2, 8, torch.device("cuda", 0))
    got = paged.build_tables(lens, i32([1, 2]), t, f, n_free, page_size=16, max_tokens=8, out=out)
    assert got is out and out.lens.tolist() == [6, 2]
    with pytest.raises(Exception, match="overlaps"):
        paged.build_tables(out.lens, i32([1, 1]), t, f, out.n_free, page_size=16, max_tokens=8, out=out)
    with pytest.raises(ValueError, match="shape"):
        paged.build_tables(lens, i32([1]), t, f, n_free, page_size=16, max_tokens=8)
    with pytest.raises(ValueError, match="page_size"):
        paged.build_tables(lens, i32([1, 1]), t, f, n_free, page_size=20, max_tokens=8)


# ---- append and gather -----------------------------------------------------------
def _edge_rows(dtype, n, dh, seed):
    """Rows with what a quantizer meets: smooth values, grids whose quotients
    end at a half, zeros, constants, one sign, tiny and huge ones, an outlier."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, dh, generator=g)
    for i in range(n):
        k = i % 10
        if k == 1:
            x[i] = torch.arange(dh) % 31 * 0.5 - 7
        elif k == 2:
            x[i] = 0
        elif k == 3:
            x[i] = -2.5
        elif k == 4:
            x[i] = x[i].abs() + 50
        elif k == 5:
            x[i] *= 2.0 ** -13
        elif k == 6:
            x[i] *= 15000
        elif k == 7:
            x[i, i % dh] = 1000
        elif k == 8:
            x[i] = -x[i].abs()
        elif k == 9:
            x[i] = (torch.arange(dh) % 16) / 15
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dh, group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("n, hkv, page, layout", [
    (1, 1, 16, "plain"), (17, 3, 16, "packed"), (40, 2, 64, "odd"), (333, 1, 128, "heads"), (65, 8, 32, "packed")])
def test_append_and_gather(dtype, dh, group, n, hkv, page, layout):
    pages = cdiv(n, page) + 2
    pools, want = [], []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        pools += [torch.randint(-2 ** 31, 2 ** 31, (pages, hkv, page, dh // 8), generator=g).int().cuda(),
                  torch.randn(pages, hkv, page, dh // group, generator=g).to(dtype).cuda(),
                  torch.randn(pages, hkv, page, dh // group, generator=g).to(dtype).cuda()]
    want = [p.clone() for p in pools]
    slots = torch.randperm(pages * page)[:n]
    slots[3::7] = -1
    if n > 5:
        slots[5] = pages * page                  # just past the pool
    rows = [_edge_rows(dtype, n * hkv, dh, s).view(n, hkv, dh) for s in (3, 4)]
    if layout == "plain":
        kv = [r.cuda() for r in rows]
    elif layout == "packed":
        qkv = torch.zeros(n, 3 * hkv, dh, dtype=dtype, device="cuda")
        qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:] = rows[0].cuda(), rows[1].cuda()
        kv = [qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:]]
    elif layout == "heads":
        kv = [r.transpose(0, 1).contiguous().cuda().transpose(0, 1) for r in rows]
    else:                                        # rows that start at any element
        kv = []
        for r in rows:
            buf = torch.zeros(n * (hkv * dh + 3) + 1, dtype=dtype, device="cuda")
            view = buf[1:].as_strided((n, hkv, dh), (hkv * dh + 3, dh, 1), 1)
            view.copy_(r)
            kv.append(view)
    for half in range(2):
        codes, s, z = quant.canonical_quantize(rows[half].reshape(-1, dh).numpy(), 4, group)
        w = torch.from_numpy(quant.pack_codes(codes, 4).view(np.int32))
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                at = (slot // page, slice(None), slot % page)
                sl = slice(i * hkv, (i + 1) * hkv)
                want[3 * half][at] = w[sl].cuda()
                want[3 * half + 1][at] = torch.from_numpy(s[sl]).cuda()
                want[3 * half + 2][at] = torch.from_numpy(z[sl]).cuda()
    ts = slots.cuda()
    paged.append(*kv, *pools, ts)
    for got, w in zip(pools, want):
        assert torch.equal(got, w)
    for out_dtype in {dtype, F32}:
        for half, got in enumerate(paged.gather(*pools, ts, dtype=out_dtype)):
            live = (slots >= 0) & (slots < pages * page)
            assert got.dtype == out_dtype and bool((got[~live.cuda()] == 0).all())
            at = ts[live.cuda()]
            rows_ = [p[at // page, :, at % page].cpu() for p in pools[3 * half:3 * half + 3]]
            m = rows_[0].shape[0] * hkv
            codes = quant.unpack_codes(rows_[0].reshape(m, -1).numpy().view(np.uint32), 4, dh)
            vals = quant.dequantize(codes, rows_[1].reshape(m, -1).numpy(), rows_[2].reshape(m, -1).numpy(),
                                    group, np.float32)
            assert torch.equal(got[live.cuda()].cpu(), torch.from_numpy(vals).view(-1, hkv, dh).to(out_dtype))


def test_append_of_nothing_and_refusals():
    p = [torch.zeros(2, 2, 16, 16, dtype=torch.int32, device="cuda"),
         *(torch.zeros(2, 2, 16, 2, dtype=F16, device="cuda") for _ in range(2))] * 2
    x = torch.zeros(0, 2, 128, dtype=F16, device="cuda")
    slots = torch.zeros(0, dtype=torch.int64, device="cuda")
    paged.append(x, x, *p, slots)
    assert paged.gather(*p, slots)[0].shape == (0, 2, 128)
    x, slots = torch.zeros(3, 2, 128, dtype=F16, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad, match in ((dict(keys=x.float()), "holds"), (dict(values=x[:2]), "shape"),
                       (dict(slots=slots.int()), "int32"), (dict(keys=x.cpu()), "cpu"),
                       (dict(keys=torch.zeros(3, 2, 256, dtype=F16, device="cuda")[..., ::2]), "contiguous")):
        kw = dict(keys=x, values=x, slots=slots) | bad
        with pytest.raises(ValueError, match=match):
            paged.append(kw["keys"], kw["values"], *p, kw["slots"])
    with pytest.raises(ValueError, match="float32"):
        paged.gather(*p, slots, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="contiguous"):
        paged.gather(p[0].transpose(0, 1), *p[1:], slots)
    with pytest.raises(Exception, match="16-byte"):
        off = torch.zeros(2 * 2 * 16 * 16 + 1, dtype=torch.int32, device="cuda")[1:].view(2, 2, 16, 16)
        paged.gather(off, *p[1:], slots)


# ---- attention -----------------------------------------------------------------
# ctx, new, hkv, r, dh, group, page, dtype
ATTEND = [
    ([0], [1], 1, 1, 128, 64, 16, F16), ([1], [1], 1, 4, 128, 64, 16, F16),
    ([15], [1], 2, 4, 128, 64, 16, F16), ([16], [1], 2, 4, 64, 64, 16, F16), ([17], [1], 2, 8, 128, 128, 32, F16),
    ([127, 128, 129], [1, 1, 1], 2, 7, 128, 32, 64, F16), ([1000], [1], 8, 4, 128, 64, 64, F16),
    ([5000, 3, 0, 777], [1, 1, 1, 1], 4, 3, 128, 64, 128, F16), ([2049] * 5, [1] * 5, 1, 16, 64, 32, 16, F16),
    ([40000], [1], 2, 8, 128, 64, 64, F16), ([300] * 70, [1] * 70, 1, 5, 128, 64, 16, F16),
    ([100, 0, 33], [2, 3, 4], 2, 4, 128, 64, 16, F16), ([513, 64], [4, 1], 8, 2, 64, 64, 32, F16),
    ([100, 0, 33, 2000], [5, 0, 8, 7], 2, 4, 128, 64, 16, F16), ([9, 200], [9, 16], 2, 7, 128, 128, 16, F16),
    ([0], [64], 1, 4, 128, 64, 16, F16), ([0, 0], [128, 129], 2, 2, 128, 64, 16, F16),
    ([777], [200], 2, 4, 128, 64, 64, F16), ([130, 4000, 0, 1], [31, 1, 300, 77], 2, 4, 128, 64, 16, F16),
    ([64, 65], [33, 500], 1, 8, 64, 32, 32, F16), ([1024], [1024], 1, 1, 128, 128, 128, F16),
    ([333, 100], [150, 17], 1, 3, 64, 64, 16, F16), ([200], [90], 1, 33, 128, 64, 16, F16),
    ([10, 2500], [600, 40], 2, 5, 128, 32, 16, F16), ([0, 5, 9], [0, 0, 0], 1, 2, 128, 64, 16, F16),
    ([0], [1], 1, 1, 64, 32, 16, F32), ([77, 3001], [1, 1], 2, 3, 64, 32, 16, F32),
    ([500, 0, 31], [3, 5, 2], 2, 4, 128, 64, 32, F32), ([256], [70], 1, 2, 128, 128, 64, F32),
    ([6000], [1], 1, 8, 128, 64, 128, F32), ([40, 41], [17, 1], 4, 1, 64, 64, 16, F32),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "ctx%s-new%s-%dx%d-dh%d-g%d-p%d-%s" % (
    "_".join(map(str, c[0][:4])), "_".join(map(str, c[1][:4])), *c[2:7], str(c[7])[6:]))
def test_attend(case):
    s = Step(*case, seed=len(case[0]))
    s.check(s.call(paged))


@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_reads_any_stride_and_leaves_padding(new, dtype):
    """Contiguous, packed and oddly aligned rows, loose bounds, padded tokens."""
    s = Step([100, 37], [new, 1], 2, 3, 128, 64, 16, dtype, pad=5, packed=False, extra_width=3)
    s.check(s.call(paged))
    for name in ("q", "nk", "nv"):
        x = getattr(s, name)
        n, h, d = x.shape
        buf = torch.zeros(n * h * (d + 1) + 9, dtype=dtype, device="cuda")
        view = buf.as_strided((n, h, d), (h * (d + 1), d + 1, 1), 3)
        view.copy_(x)
        setattr(s, name, view)
    out = torch.full((new + 6, 6, 128), 7.0, dtype=dtype, device="cuda")
    got = s.call(paged, out=out, max_ctx=None, max_new=new + 40)
    assert got is out
    s.check(got)
    assert bool((out[new + 1:] == 7.0).all())


@pytest.mark.parametrize("layout", ["plain", "packed", "heads", "one head for all", "odd"])
@pytest.mark.parametrize("dh, hkv, r", [(128, 2, 4), (64, 3, 1), (128, 1, 2)])
def test_attend_long_own_entries_of_any_layout(layout, dh, hkv, r):
    """Whole tiles of the step's own keys and values, whatever their strides,
    behind another request's; a NaN behind the last request's tokens."""
    s = Step([30, 0, 200], [3, 700, 390], hkv, r, dh, 64, 16, F16, pad=200, packed=layout == "packed")
    for name in ("nk", "nv"):
        x = getattr(s, name)
        x[1093:] = float("nan")
        if layout == "heads":
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        elif layout == "one head for all":
            x = x[:, :1].expand(-1, hkv, -1)
        elif layout == "odd":
            buf = torch.zeros(x.numel() + x.shape[0] + 1, dtype=F16, device="cuda")
            view = buf.as_strided(x.shape, (hkv * dh + 1, dh, 1), 1)
            view.copy_(x)
            x = view
        setattr(s, name, x)
    s.check(s.call(paged))


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("spread", [1e-3, 0.03, 6.0])
def test_attend_small_and_peaky_values(new, spread):
    """Values near float16's small end keep their relative precision; large
    ones make a softmax of a single weight."""
    s = Step([700], [new], 1, 4, 128, 64, 16, F16, spread=spread)
    s.check(s.call(paged))


@pytest.mark.parametrize("new", [1, 70])
def test_attend_value_scales_far_apart(new):
    """One position's scale 2^13 times the others' does not cost them theirs."""
    s = Step([600], [new], 1, 4, 128, 64, 16, F16)
    page = int(s.tables[0, 20])
    s.pools[4][page, 0, 3] *= 2.0 ** 13
    s.pools[5][page, 0, 3] *= 2.0 ** 13
    s.check(s.call(paged))


@pytest.mark.parametrize("new", [1, 2, 70])
def test_attend_bad_pages_are_not_read(new):
    """A page id outside the pool: NaN for the request that needs it, the
    others' rows as ever."""
    for bad in (-1, 1 << 30, -2 ** 31):
        s = Step([50, 200, 90], [new, new, 1], 2, 4, 128, 64, 16, F16)
        s.tables[1, 5] = bad
        got = s.call(paged)
        cu = s.cu.tolist()
        assert bool(torch.isnan(got[cu[1]:cu[2]]).all())
        s.tables[1, 5] = 0
        s.pools[1].nan_to_num_(0), s.pools[2].nan_to_num_(0), s.pools[4].nan_to_num_(0), s.pools[5].nan_to_num_(0)
        want, tol = s.reference()
        for lo, hi in ((0, cu[1]), (cu[2], cu[3])):
            assert bool(((got[lo:hi].double() - want[lo:hi]).abs() <= tol[lo:hi]).all())


@pytest.mark.parametrize("new, at", [(4, 2), (200, 130), (200, 3)])
@pytest.mark.parametrize("what", ["nk", "nv"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attend_keeps_later_tokens_out(new, at, what, value):
    """A NaN or an infinity in an own entry reaches the tokens that see it and
    none before it, nor another request."""
    s = Step([60, 50], [new, 3], 2, 4, 128, 64, 16, F16, packed=False)
    want, tol = s.reference()
    getattr(s, what)[at, 1, 17] = value
    got = s.call(paged)
    off = (got.double() - want).abs() <= tol
    assert bool(off[:at].all()) and bool(off[new:].all()) and bool(off[:new, :4].all())
    if what == "nv" or value != value:
        assert bool((~torch.isfinite(got[at:new, 4:])).any(-1).all())


@pytest.mark.parametrize("new, r", [([4, 3, 1], 4), ([8, 7, 2], 4), ([1, 1, 1], 16), ([2, 1, 2], 16), ([6, 5, 1], 4),
                                    ([3, 6, 1], 5), ([32, 9, 30], 1), ([8, 90, 9], 4), ([1, 50, 2], 32), ([2, 33, 1], 48)])
@pytest.mark.parametrize("loose", [False, True])
def test_attend_columns_per_pass(new, r, loose):
    """Few columns in one pass or several, tiles of eight or, where the bounds
    allow long caches, sixteen; beside chunks and alone."""
    s = Step([200, 75, 16], new, 2, r, 128, 64, 16, F16, extra_width=60000 if loose else 0)
    s.check(s.call(paged, max_ctx=None))


@pytest.mark.parametrize("new", [1, 70])
def test_attend_cuts_to_its_bounds(new):
    """Lengths past max_ctx and negative ones are cut, not followed."""
    s = Step([64, 30], [new, new], 1, 4, 128, 64, 16, F16)
    s.ctx_t.copy_(i32([10 ** 9, -5]))
    got = s.call(paged)
    s.ctx = [64, 0]
    s.check(got)


def test_attend_equals_the_contiguous_step():
    """One new token over one page run: `kv_attention.decode`'s result, within
    both kernels' output rounding."""
    s = Step([256], [1], 2, 4, 128, 64, 64, F16)
    order = s.tables[0, :4].long()
    flat = [p[order].transpose(0, 1).reshape(2, 256, -1).contiguous() for p in s.pools]
    want = kva.decode(s.q.contiguous(), *flat, s.nk.contiguous(), s.nv.contiguous(), bits=4)
    got = s.call(paged)
    s.check(got)
    assert float((got.float() - want.float()).abs().max()) <= 2 * 2.0 ** -10 * float(want.abs().max())


def test_attend_is_repeatable_and_streams_do_not_share():
    """The same bits every time, also with calls in flight on several streams."""
    steps = [Step([3000, 50], [1, 1], 4, 4, 128, 64, 64, F16, seed=i) for i in range(3)] + \
            [Step([500], [300], 4, 4, 128, 64, 64, F16, seed=9)]
    want = [s.call(paged).clone() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[] for _ in steps]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(steps, streams)):
            got[i].append(s.call(paged, stream=st))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@pytest.mark.parametrize("case", [([60, 50], [200, 3], 2, 4), ([700, 0, 33], [130, 64, 9], 4, 2), ([300], [5], 8, 8)])
def test_attend_same_bits_many_times(case):
    """Short units of several lengths behind one another in every CTA's share,
    call after call: a buffer taken over too early shows as a differing bit."""
    s = Step(*case, 128, 64, 16, F16, packed=False)
    want = s.call(paged).clone()
    s.check(want)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        differ += (s.call(paged) != want).sum()
    assert differ.item() == 0


def test_attend_captured_step_follows_lengths():
    """One captured step replayed for other lengths within its bounds, beside
    a second graph of the same tensors."""
    s = Step([700, 300, 90], [3, 1, 40], 2, 4, 128, 64, 16, F16)
    s.call(paged)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.call(paged))
        graphs.append(g)
    for ctx, new in (([700, 300, 90], [3, 1, 40]), ([1, 299, 90], [1, 1, 1]), ([650, 0, 17], [40, 0, 4])):
        s.ctx, s.new = ctx, new
        s.ctx_t.copy_(i32(ctx))
        s.cu.copy_(i32([sum(new[:i]) for i in range(4)]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        n = sum(new)
        want, tol = s.reference()
        for out in outs:
            assert bool(((out[:n].double() - want[:n]).abs() <= tol[:n]).all())
    del graphs


def test_attend_captured_chunk_reads_its_tensors_anew():
    """A captured chunk with whole tiles of own entries, replayed over other
    queries, keys and values in the same memory."""
    s = Step([100, 20], [400, 2], 2, 4, 128, 64, 16, F16)
    s.call(paged)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.call(paged)
    g = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(2):
        for x in (s.q, s.nk, s.nv):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        s.check(out)
    del graph


def test_attend_refusals():
    s = Step([20], [2], 2, 2, 128, 64, 16, F16)
    ok = dict(block_tables=s.tables, ctx_lens=s.ctx_t, cu_new=s.cu, max_new=2)

    def call(q=s.q, nk=s.nk, nv=s.nv, pools=s.pools, **over):
        return paged.attend(q, *pools, nk, nv, **(ok | over))

    for bad, match in ((dict(q=s.q[:, :3]), "divide"), (dict(q=s.q.float()), "holds"), (dict(nk=s.nk[:1]), "shape"),
                       (dict(cu_new=s.cu[:1]), "shape"), (dict(ctx_lens=s.ctx_t.long()), "int64"),
                       (dict(max_ctx=10 ** 6), "max_ctx"), (dict(max_new=-1), "max_new"),
                       (dict(block_tables=s.tables.t()), "shape|contiguous"), (dict(out=s.q), "contiguous"),
                       (dict(q=s.q.cpu()), "cpu"), (dict(pools=s.pools[:3] + [p.float() for p in s.pools[3:]]), "int32|float")):
        with pytest.raises(ValueError, match=match):
            call(**bad)
    assert call(max_new=0).shape == s.q.shape            # nothing to do, nothing written


# ---- a serving step of all of them ---------------------------------------------
@pytest.mark.parametrize("dtype", [F16, F32])
def test_serving_steps(dtype):
    """Requests of several lengths admitted, extended, cut back and ended over
    one pool; every step's attention against 64 bits over what the cache
    holds, every page accounted for."""
    rows, hkv, r, dh, group, page, pages, width = 4, 2, 4, 128, 64, 16, 60, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    pools = []
    for _ in range(2):
        pools += [torch.zeros(pages, hkv, page, dh // 8, dtype=torch.int32, device="cuda"),
                  *(torch.full((pages, hkv, page, dh // group), float("nan"), dtype=dtype, device="cuda")
                    for _ in range(2))]
    tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages).int().cuda()
    lens, n_free = i32([0] * rows), i32([pages])
    for new, keep in (([40, 1, 0, 130], None), ([1, 1, 90, 1], None), ([4, 3, 1, 2], [43, 4, 91, 133]),
                      ([1, 1, 1, 1], [0, 5, 92, 0]), ([200, 1, 1, 33], None), ([1, 1, 1, 1], None)):
        b = paged.build_tables(lens, i32(new), tables, free, n_free, page_size=page, max_tokens=260)
        assert b.status.item() == 0
        qkv = torch.randn(260, hkv * (r + 2), dh, generator=g, device="cuda").to(dtype)
        s = Step.__new__(Step)
        s.ctx, s.new, s.hkv, s.r, s.dh, s.group, s.page, s.dtype = lens.tolist(), new, hkv, r, dh, group, page, dtype
        s.q, s.nk, s.nv = qkv[:, :hkv * r], qkv[:, hkv * r:hkv * (r + 1)], qkv[:, hkv * (r + 1):]
        s.pools, s.tables, s.ctx_t, s.cu = pools, tables, lens, b.cu_new
        paged.append(s.nk, s.nv, *pools, b.slots)        # the step's rows are past ctx: not read by it
        s.check(s.call(paged, max_new=260, max_ctx=None))
        lens, n_free = b.lens, b.n_free
        if keep is not None:
            lens, n_free = paged.truncate(lens, i32(keep), tables, free, n_free, page_size=page)
        held = [int(x) for t, n in zip(tables.tolist(), lens.tolist()) for x in t[:cdiv(n, page)]]
        assert sorted(held + free.tolist()[:n_free.item()]) == list(range(pages))
