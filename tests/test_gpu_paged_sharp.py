"""The paged attention against 64 bits under a bound that a lost or doubled run
of positions breaks: every block of a cache in turn, batches of more requests
than the kernels have threads, contexts from one position to long ones."""

from __future__ import annotations

import random

import pytest
import torch

from kernelverify_b200.pack import paged
from tests import paged_sharp as sharp
from tests.paged_cases import Step, cdiv
from tests.test_gpu_paged import ATTEND, i32

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _needs(native):
    torch.manual_seed(0)


@pytest.mark.parametrize("case", [c for c in ATTEND if sum(c[1])], ids=lambda c: "ctx%s-new%s-%dx%d-dh%d-g%d-p%d-%s" % (
    "_".join(map(str, c[0][:4])), "_".join(map(str, c[1][:4])), *c[2:7], str(c[7])[6:]))
def test_attend(case):
    s = Step(*case, seed=len(case[0]))
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("ctx, new, hkv, r, dh, group, page, dtype", [
    (5000, 1, 2, 4, 128, 64, 16, F16), (5000, 1, 1, 2, 64, 32, 32, F16), (3000, 3, 2, 4, 128, 64, 16, F16),
    (2500, 4, 2, 4, 128, 128, 64, F16), (1000, 9, 2, 4, 128, 64, 16, F16), (1700, 40, 1, 4, 128, 64, 16, F16),
    (900, 130, 1, 2, 64, 64, 16, F16), (2500, 1, 2, 4, 128, 64, 16, F32), (900, 5, 1, 3, 64, 32, 16, F32)])
def test_every_block_counts_once(ctx, new, hkv, r, dh, group, page, dtype):
    """64 requests of about ctx positions, each (request, cache head) with half of its
    weight on one block of 16 and values nowhere else; each block is somewhere."""
    lens = [ctx - 3 * b for b in range(64)]
    s = Step(lens, [new] * 64, hkv, r, dh, group, page, dtype, packed=False)
    last = [cdiv(n, 16) - 1 for n in lens]
    order = list(range(last[0] + 1))
    random.Random(ctx).shuffle(order)
    order *= cdiv(64 * hkv, len(order)) + 1
    for at in range(0, last[0] + 1, 64 * hkv):
        blocks = [[min(order[at + b * hkv + h], last[b]) for h in range(hkv)] for b in range(64)]
        sharp.mark(s, blocks)
        sharp.check(s, s.call(paged))


@pytest.mark.parametrize("ctx, new, hkv, r, dtype", [(40000, 1, 2, 8, F16), (70001, 1, 1, 4, F16), (40000, 2, 1, 8, F16),
                                                     (20000, 300, 1, 4, F16), (20000, 1, 1, 4, F32)])
def test_blocks_of_a_long_sequence(ctx, new, hkv, r, dtype):
    """One sequence over all CTAs: its first, last and 24 other blocks."""
    s = Step([ctx], [new], hkv, r, 128, 64, 64, dtype, packed=False)
    last = cdiv(ctx, 16) - 1
    rng = random.Random(ctx)
    for at in [0, last] + [rng.randrange(last) for _ in range(24)]:
        sharp.mark(s, [[at] * hkv])
        sharp.check(s, s.call(paged))


@pytest.mark.parametrize("new", [200, 600])
def test_own_entries_of_a_chunk_count_once(new):
    """Half of the weight of the last token on one of the chunk's own entries, the
    values zero elsewhere."""
    s = Step([130], [new], 1, 4, 128, 64, 16, F16, packed=False)
    sharp.mark(s, [[0]])
    for t in s.pools[2], s.pools[4], s.pools[5]:
        t.zero_()
    for at in sorted({0, 1, 63, 64, 65, 127, 128, 129, 191, new // 2, new - 2, new - 1}):
        s.nk.zero_(), s.nv.zero_()
        s.nk[at], s.nv[at] = 0.5, 0.75
        sharp.check(s, s.call(paged))


@pytest.mark.parametrize("r", [64, 65, 100, 128, 129, 200])
@pytest.mark.parametrize("ctx, new", [([300, 5], [1, 1]), ([130, 0, 40], [7, 3, 1]), ([257], [150])])
def test_many_query_heads(ctx, new, r):
    """One token, or half of one, to a tile of queries."""
    s = Step(ctx, new, 1, r, 64, 64, 16, F16)
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("rows", [600, 4096])
@pytest.mark.parametrize("new, dtype", [((1, 1), F16), ((0, 3), F16), ((0, 12), F16), ((1, 2), F32)])
def test_attend_many_requests(rows, new, dtype):
    """More requests than a kernel has threads: each thread sums several rows'
    tiles."""
    rng = random.Random(rows)
    ctx = [rng.choice([0, 1, 15, 16, 33, 70]) for _ in range(rows)]
    s = Step(ctx, [rng.randint(*new) for _ in range(rows)], 1, 4, 64, 64, 16, dtype, packed=False)
    got = s.call(paged)
    picked = sorted(rng.sample(range(rows), 60) + [0, rows - 1])
    _check_rows(s, got, picked)
    assert bool(torch.isfinite(got[:sum(s.new)]).all())


def test_attend_many_requests_beside_chunks():
    """Both kernels over a batch of 4096 rows, most of them empty."""
    rng = random.Random(1)
    rows = 4096
    ctx, new = [0] * rows, [0] * rows
    for b in rng.sample(range(rows), 200):
        ctx[b], new[b] = rng.randint(0, 200), rng.choice([1, 1, 2, 30, 90])
    s = Step(ctx, new, 1, 4, 128, 64, 16, F16, packed=False)
    _check_rows(s, s.call(paged), [b for b in range(rows) if new[b]])


def _check_rows(s, got, picked):
    """sharp.check of some of the requests (each reference is a few small products)."""
    cu = s.cu.tolist()
    for b in picked:
        if s.new[b] == 0:
            continue
        t = Step.__new__(Step)
        t.__dict__.update(s.__dict__)
        lo, hi = cu[b], cu[b + 1]
        t.ctx, t.new = [s.ctx[b]], [s.new[b]]
        t.q, t.nk, t.nv = s.q[lo:hi], s.nk[lo:hi], s.nv[lo:hi]
        t.tables, t.cu = s.tables[b:b + 1], i32([0, hi - lo])
        sharp.check(t, got[lo:hi])


@pytest.mark.parametrize("new", [1, 6, 70])
@pytest.mark.parametrize("spread", [1e-3, 0.03, 6.0])
def test_small_and_peaky_values(new, spread):
    s = Step([700], [new], 1, 4, 128, 64, 16, F16, spread=spread)
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("new, dtype", [(1, F16), (6, F16), (70, F16), (1, F32)])
def test_values_beside_an_outlier(new, dtype):
    """One position's scale 2^13 times the others' does not cost them theirs, seen
    where its code stands for zero."""
    s = Step([600], [new], 1, 4, 128, 64, 16, dtype)
    sharp.outlier(s, 0, 0, 323)
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("ctx", [1, 2, 5, 16, 17, 40, 256])
@pytest.mark.parametrize("new", [1, 4, 80])
def test_short_contexts(ctx, new):
    """Where nothing averages the roundings."""
    s = Step([ctx, ctx + 1], [new, 1], 2, 4, 128, 64, 16, F16)
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("ctx", [1, 2, 4, 8, 32, 100, 256])
@pytest.mark.parametrize("new, r, dh", [(1, 4, 128), (1, 8, 64), (4, 4, 128)])
def test_short_contexts_are_rounded_once(ctx, new, r, dh):
    """Requests with few tokens and few cached positions: the error is the output's
    own rounding (root mean squares within a tenth: other roundings of half its size
    would add an eighth), weights rounded to float16 would add up to two fifths."""
    own = err = 0.0
    for seed in range(8):
        s = Step([ctx] * 4, [new] * 4, 2, r, dh, 64, 16, F16, seed=seed, packed=False)
        want = sharp.reference(s)[0]
        err += float((s.call(paged).double() - want).square().sum())
        own += float((want.half().double() - want).square().sum())
    assert err <= 1.1 ** 2 * own


def test_a_captured_step_over_other_lengths():
    s = Step([700, 300, 90], [3, 1, 40], 2, 4, 128, 64, 16, F16)
    s.call(paged)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = s.call(paged)
    for ctx, new in (([700, 300, 90], [3, 1, 40]), ([1, 299, 90], [1, 1, 1]), ([650, 0, 17], [40, 0, 4])):
        s.ctx, s.new = ctx, new
        s.ctx_t.copy_(i32(ctx))
        s.cu.copy_(i32([sum(new[:i]) for i in range(4)]))
        g.replay()
        n = sum(new)
        want, sigma, drift = sharp.reference(s)
        err = (out[:n].double() - want[:n]).abs()
        assert bool((err <= 8 * sigma[:n] + drift[:n]).all())
    del g
