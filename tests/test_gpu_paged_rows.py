"""Append and read-back of the paged cache at the ends of what they accept."""

from __future__ import annotations

import pytest
import torch

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
