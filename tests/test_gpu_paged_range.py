"""The paged attention at the ends of its values' range: infinite keys of either
sign among the step's own entries, and float32 steps up to 2^60."""

from __future__ import annotations

import pytest
import torch

from kernelverify_b200.pack import paged
from tests import paged_sharp as sharp
from tests.paged_cases import Step

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _needs(native):
    torch.manual_seed(0)


@pytest.mark.parametrize("dtype, new, at", [(F16, 4, 2), (F16, 200, 130), (F16, 200, 3), (F16, 1, 0), (F32, 5, 2)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_an_infinite_key(dtype, new, at, value):
    """A score of +inf makes the rows that see it not finite; one of -inf takes the
    entry out of them. Rows before it, other heads and requests are as ever."""
    s = Step([60, 50], [new, 3], 2, 4, 128, 64, 16, dtype, packed=False)
    heads, dim = torch.arange(4, device="cuda") + s.r, 17             # of cache head 1
    sign = torch.tensor([1.0, -1.0, 0.5, -2.0], device="cuda")
    s.q[:, heads, dim] = sign.to(dtype)
    want, sigma, drift = sharp.reference(s)
    s.nk[at, 1] = 0
    s.nk[at, 1, dim] = 2000.0 if value > 0 else -2000.0               # a score of 88 or more either way
    gone, gone_sigma, gone_drift = sharp.reference(s)
    s.nk[at, 1, dim] = value
    got = s.call(paged)

    def within(rows, want, sigma, drift):
        return bool(((got.double() - want).abs() <= 8 * sigma + drift)[rows].all())
    assert within(slice(0, at), want, sigma, drift) and within(slice(new, None), want, sigma, drift)
    assert within((slice(0, new), slice(0, s.r)), want, sigma, drift)
    high = (sign * value > 0).tolist()
    for h, up in zip(heads.tolist(), high):
        if up:
            assert bool((~torch.isfinite(got[at:new, h])).any(-1).all())
        else:
            assert within((slice(at, new), h), gone, gone_sigma, gone_drift)


@pytest.mark.parametrize("ctx, new, r", [([300], [1], 4), ([40, 0], [5, 3], 2), ([700], [60], 1)])
@pytest.mark.parametrize("exponent", [-19, 59])
def test_float32_values_up_to_their_limits(ctx, new, r, exponent):
    """Values near 2^60, and scales near the quantizer's smallest step, 1e-7, with the
    relative precision of others."""
    s = Step(ctx, new, 2, r, 128, 64, 16, F32, packed=False)
    for t in (s.nv, s.pools[4], s.pools[5]):
        t.mul_(2.0 ** exponent / 8)
    sharp.check(s, s.call(paged))


@pytest.mark.parametrize("ctx, new, r", [([300], [1], 4), ([40, 0], [5, 3], 2), ([700], [60], 1)])
@pytest.mark.parametrize("exponent", [-57, -40, 40, 57])
def test_float32_queries_of_any_size(ctx, new, r, exponent):
    """Queries of any size against keys that are smaller by as much."""
    s = Step(ctx, new, 2, r, 128, 64, 16, F32, packed=False)
    s.q.mul_(2.0 ** exponent)
    for t in (s.nk, s.pools[1], s.pools[2]):
        t.mul_(2.0 ** -exponent)
    sharp.check(s, s.call(paged))
