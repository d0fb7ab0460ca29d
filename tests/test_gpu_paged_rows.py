"""Append and read-back of the paged cache at the ends of what they accept."""

from __future__ import annotations

import pytest
import torch

from kernelverify_b200.pack import kv_attention as kva
from kernelverify_b200.pack import paged

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _needs(native):
    torch.manual_seed(0)


def pool(pages, heads, page, dh, group, dtype):
    return [torch.zeros(pages, heads, page, dh // 8, dtype=torch.int32, device="cuda"),
            *(torch.zeros(pages, heads, page, dh // group, dtype=dtype, device="cuda") for _ in range(2))]


def test_append_refuses_arrays_over_one_another():
    k, v = pool(2, 2, 16, 128, 64, F16), pool(2, 2, 16, 128, 64, F16)
    x = torch.randn(3, 2, 128, device="cuda").to(F16)
    slots = torch.arange(3, device="cuda")
    inside = k[0].view(F16).view(-1)[:3 * 2 * 128].view(3, 2, 128)
    for keys, values, kp, vp, at in ((x, x, k, k, slots), (x, x, k, [v[0], v[1], k[2]], slots),
                                     (x, x, k, [v[0], v[1], v[1]], slots), (inside, x, k, v, slots),
                                     (x, inside, k, v, slots), (x, x, k, v, v[0].view(-1)[:6].view(torch.int64))):
        with pytest.raises(Exception, match="overlaps"):
            paged.append(keys, values, *kp, *vp, at)
    assert all(bool((t == 0).all()) for t in k + v)
    paged.append(x, x, *k, *v, slots)                  # keys and values may be one tensor
    assert all(torch.equal(a, b) for a, b in zip(k, v))
    got = paged.gather(*k, *k, slots)                  # and one pool may be read twice
    assert torch.equal(*got)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dh, group", [(64, 32), (128, 64), (128, 128)])
def test_append_of_what_is_not_finite(dtype, dh, group):
    """NaN and infinities, and in float32 groups whose range is infinite: the bits
    of the other quantizer."""
    top = torch.finfo(dtype).max
    inf, nan = float("inf"), float("nan")
    rows = torch.randn(16, 1, dh)
    for i, values in enumerate(([nan], [inf], [-inf], [inf, -inf], [nan, inf], [nan, -inf], [nan] * dh, [inf] * dh,
                                [-inf] * dh, [top, -top], [-top, top / 2], [top], [-top], [0.0, -0.0] * (dh // 2),
                                [torch.finfo(dtype).tiny], [1e-7, -1e-7, nan])):
        rows[i, 0, :len(values)] = torch.tensor(values)
    x = rows.to(dtype).cuda()
    k, v = pool(1, 1, 16, dh, group, dtype), pool(1, 1, 16, dh, group, dtype)
    slots = torch.arange(16, device="cuda")
    paged.append(x, x.neg(), *k, *v, slots)
    for got, values in ((k, x), (v, x.neg())):
        words, scales, biases = kva.quantize_cache(values.transpose(0, 1).contiguous(), bits=4, group_size=group)
        assert torch.equal(got[0][0].view(torch.int32), words.view(torch.int32))
        for a, b in ((got[1][0], scales), (got[2][0], biases)):
            assert torch.equal(a.isnan(), b.isnan())
            assert torch.equal(a.nan_to_num(0.0, inf, -inf), b.nan_to_num(0.0, inf, -inf))


@pytest.mark.parametrize("rows, cut, room", [(3, 4, 5), (3, 4, 12), (3, 4, 0), (40, 7, 100)])
def test_truncate_into_a_stack_without_room(rows, cut, room):
    """What does not fit on the stack is dropped; nothing behind it is written."""
    page, held = 16, cut + 2
    tables = torch.arange(rows * held, dtype=torch.int32, device="cuda").view(rows, held)
    lens = torch.full((rows,), held * page - 3, dtype=torch.int32, device="cuda")
    keep = torch.full((rows,), 2 * page, dtype=torch.int32, device="cuda")
    stack = 6
    buf = torch.full((stack + room + 50,), -9, dtype=torch.int32, device="cuda")
    free, n_free = buf[:stack + room], torch.tensor([stack], dtype=torch.int32, device="cuda")
    out = torch.full((rows,), -1, dtype=torch.int32, device="cuda"), torch.full((1,), -1, dtype=torch.int32, device="cuda")
    got = paged.truncate(lens, keep, tables, free, n_free, page_size=page, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    back = tables[:, 2:].flatten().tolist()[:room]
    assert out[0].tolist() == [2 * page] * rows and out[1].item() == stack + len(back)
    assert buf.tolist() == [-9] * stack + back + [-9] * (buf.numel() - stack - len(back))
    with pytest.raises(ValueError, match="out"):
        paged.truncate(lens, keep, tables, free, n_free, page_size=page, out=(out[0][:-1], out[1]))
    with pytest.raises(ValueError, match="out"):
        paged.truncate(lens, keep, tables, free, n_free, page_size=page, out=(out[0].long(), out[1]))


@pytest.mark.parametrize("dh, group", [(64, 32), (128, 64)])
@pytest.mark.parametrize("exponent", [-149, -130, -126, -122, -20, 0, 100, 114, 118, 123])
def test_read_back_of_float32_scales_of_any_size(dh, group, exponent):
    """scale * code + bias, a rounded product and a rounded sum, at both ends of the
    scales' range: finite where the value is."""
    g = torch.Generator().manual_seed(exponent + 200)
    k = pool(2, 1, 16, dh, group, F32)
    codes = torch.randint(0, 16, (32, dh), generator=g)
    words = sum(codes[:, i::8].long() << (4 * i) for i in range(8))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    scales = torch.ldexp(torch.rand(32, dh // group, generator=g) + 1.0, torch.tensor(exponent))
    scales *= torch.where(torch.rand(32, dh // group, generator=g) < 0.5, -1.0, 1.0)
    biases = -scales * torch.randint(0, 16, (32, dh // group), generator=g)
    for t, x in zip(k, (words, scales, biases)):
        t.copy_(x.view(t.shape))
    want = (codes.float() * scales.repeat_interleave(group, 1)) + biases.repeat_interleave(group, 1)
    got, _ = paged.gather(*k, *k, torch.arange(32, device="cuda"))
    assert torch.equal(got.cpu().view(32, dh), want)
