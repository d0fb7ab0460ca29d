"""The paged cache where addresses are wide and calls overlap: pools and inputs
whose offsets pass 32 bits, every entry on a stream of its own, calls from
several host threads."""

from __future__ import annotations

import threading

import pytest
import torch

from kernelverify_b200.pack import paged
from tests.paged_cases import Step
from tests.test_gpu_paged import i32

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(autouse=True)
def _needs(native):
    torch.manual_seed(0)
    yield
    torch.cuda.empty_cache()


def test_pools_past_32_bits():
    """The last pages of pools of 2^27 rows (words of 8 GiB each): the same bits as
    from small pools, written, read back and attended over."""
    hkv, dh, group, page = 8, 128, 128, 64
    pages = (1 << 27) // (hkv * page) + 5
    lead = (pages, hkv, page)
    big = [torch.zeros(*lead, dh // 8, dtype=torch.int32, device="cuda") if i % 3 == 0 else
           torch.zeros(*lead, 1, dtype=F16, device="cuda") for i in range(6)]
    assert big[0].numel() * 4 > 1 << 33
    for new in ([1, 1], [60, 3]):
        s = Step([700, 130], new, hkv, 4, dh, group, page, F16, packed=False)
        want, small = s.call(paged), s.pools
        held = small[0].shape[0]
        for t, x in zip(big, small):
            t[pages - held:] = x
        s.pools, s.tables = big, torch.where(s.tables >= 0, s.tables + (pages - held), s.tables)
        assert torch.equal(s.call(paged), want)
        # rows into the last pages' slots, and back
        n = sum(new)
        at = torch.randperm(held * page, device="cuda")[:n]
        shift = (pages - held) * page
        paged.append(s.nk, s.nv, *big, at + shift)
        paged.append(s.nk, s.nv, *small, at)
        for t, x in zip(big, small):
            assert torch.equal(t[pages - held:].nan_to_num(0) if t.is_floating_point() else t[pages - held:],
                               x.nan_to_num(0) if x.is_floating_point() else x)
        for a, b in zip(paged.gather(*big, at + shift), paged.gather(*small, at)):
            assert torch.equal(a, b)
    assert all(bool((t[:pages - held] == 0).all()) for t in big)


@pytest.mark.parametrize("new", [[1] * 9, [9], [8, 1]])
def test_rows_past_32_bits(new):
    """Tokens 2^29 + 8 elements apart: the last ones lie past 2^32 elements."""
    s = Step([100] * len(new), new, 2, 4, 128, 64, 16, F16, packed=False)
    stride = (1 << 29) + 8
    buf = torch.empty(8 * stride + 12 * 128, dtype=F16, device="cuda")
    want = s.call(paged)
    at = 0
    for name in ("q", "nk", "nv"):
        x = getattr(s, name)
        view = buf.as_strided(x.shape, (stride, 128, 1), at)
        view.copy_(x)
        setattr(s, name, view)
        at += x.shape[1] * 128
    assert torch.equal(s.call(paged), want)
    pools = [p.clone() for p in s.pools]
    slots = torch.arange(9, device="cuda") * 7
    paged.append(s.nk, s.nv, *pools, slots)
    near = [p.clone() for p in s.pools]
    paged.append(s.nk.contiguous(), s.nv.contiguous(), *near, slots)
    assert all(torch.equal(a.nan_to_num(0), b.nan_to_num(0)) if a.is_floating_point() else torch.equal(a, b)
               for a, b in zip(pools, near))


def _steps(step_of, stream):
    """A few serving steps over a small pool on `stream` (None: the current one);
    every tensor they leave."""
    rows, hkv, r, dh, group, page, pages = 3, 2, 4, 128, 64, 16, 40
    pools = [torch.zeros(pages, hkv, page, n, dtype=t, device="cuda") for n, t in
             ((dh // 8, torch.int32), (2, F16), (2, F16)) * 2]
    tables, free = torch.full((rows, 20), -1, dtype=torch.int32, device="cuda"), torch.randperm(
        pages, generator=torch.Generator().manual_seed(1)).int().cuda()
    lens, n_free = i32([0] * rows), i32([pages])
    g = torch.Generator(device="cuda").manual_seed(step_of)
    inputs = [(i32(new), i32(keep), torch.randn(150, hkv * (r + 2), dh, generator=g, device="cuda").to(F16))
              for new, keep in (([40, 1, 90], [40, 0, 90]), ([1, 1, 1], [38, 1, 91]), ([4, 100, 2], [999] * 3))]
    torch.cuda.synchronize()
    left = []
    for new, keep, qkv in inputs:
        b = paged.build_tables(lens, new, tables, free, n_free, page_size=page, max_tokens=150, stream=stream)
        q, k, v = qkv[:, :hkv * r], qkv[:, hkv * r:hkv * (r + 1)], qkv[:, hkv * (r + 1):]
        out = torch.zeros(150, hkv * r, dh, dtype=F16, device="cuda")
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        paged.append(k, v, *pools, b.slots, stream=stream)
        paged.attend(q, *pools, k, v, block_tables=tables, ctx_lens=lens, cu_new=b.cu_new, max_new=100, out=out,
                     stream=stream)
        left += [*b, out, *paged.gather(*pools, b.slots, stream=stream)]
        lens, n_free = paged.truncate(b.lens, keep, tables, free, b.n_free, page_size=page, stream=stream)
        left += [lens, n_free]
    torch.cuda.synchronize()
    return [x.clone() for x in left + [tables, free] + pools]


def test_every_entry_on_a_stream_of_its_own():
    want = _steps(5, None)
    side = torch.cuda.Stream()
    got = _steps(5, side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_from_several_threads():
    want = [_steps(i, None) for i in range(4)]
    got, errors = [[] for _ in range(4)], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            for _ in range(5):
                with torch.cuda.stream(stream):
                    got[i].append(_steps(i, None))
                with pytest.raises(Exception, match=f"page_size {17 + i}"):
                    paged.build_tables(i32([1]), i32([1]), i32([[0]]), i32([0]), i32([1]), page_size=17 + i, max_tokens=1)
        except Exception as e:                     # reported by the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for runs, w in zip(got, want):
        assert all(torch.equal(a, b) for run in runs for a, b in zip(run, w))
