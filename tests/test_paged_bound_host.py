"""The paged attention's bound itself, on the CPU: an emulation of the kernels'
roundings is within it, and outputs that lack a run of positions, or have it
twice, are not."""

from __future__ import annotations

import math

import pytest
import torch

from tests import paged_cases as pc
from tests import paged_sharp as sharp

F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _on_cpu(monkeypatch):
    monkeypatch.setattr(pc, "DEV", "cpu")


def emulated(s):
    """A kernel in float32 that rounds the weights and the cached values to
    float16 (float16 steps), 32 positions at a time under a running maximum."""
    n, h, dh = s.q.shape
    out = torch.zeros(n, h, dh)
    half = s.dtype == F16
    cu = s.cu.tolist()
    for b, length in enumerate(s.ctx):
        lo, hi = cu[b], cu[b + 1]
        for hk in range(s.hkv):
            k, _, v, _, _ = sharp.parts(s, b, hk)
            if half:
                k, v = k.half(), v.half()
            k, v = k.float(), v.float()
            for j in range(hk * s.r, (hk + 1) * s.r):
                score = s.q[lo:hi, j].float() @ k.T / math.sqrt(dh)
                score[:, length:].masked_fill_(torch.ones(hi - lo, hi - lo, dtype=torch.bool).triu(1), -math.inf)
                top = torch.full((hi - lo, 1), -math.inf)
                o, l = torch.zeros(hi - lo, dh), torch.zeros(hi - lo, 1)
                for a in range(0, k.shape[0], 32):
                    x = score[:, a:a + 32]
                    new = torch.maximum(top, x.amax(1, keepdim=True)).clamp(min=-1e30)
                    p = torch.exp(x - new)
                    o, l = o * torch.exp(top - new), l * torch.exp(top - new)
                    l = l + p.sum(1, keepdim=True)
                    o = o + ((p.half().float() if half else p) @ v[a:a + 32])
                    top = new
                out[lo:hi, j] = o / l
    return out.to(s.dtype)


CASES = [([5000, 3, 0, 777], [1, 1, 1, 1], 4, 3, 128, 64, 128, F16), ([2049] * 3, [1] * 3, 1, 16, 64, 32, 16, F16),
         ([333, 100], [150, 17], 1, 3, 64, 64, 16, F16), ([20], [3], 2, 2, 128, 64, 16, F16),
         ([6000], [1], 1, 8, 128, 64, 128, F32), ([500, 0, 31], [3, 5, 2], 2, 4, 128, 64, 32, F32)]


@pytest.mark.parametrize("case", CASES)
def test_the_roundings_are_within_the_bound(case):
    s = pc.Step(*case, seed=5)
    assert sharp.check(s, emulated(s)) <= 1.0
    assert sharp.check(s, sharp.reference(s)[0].to(s.dtype)) <= 0.5


@pytest.mark.parametrize("spread", [1e-3, 0.03, 6.0])
def test_small_and_peaky_values_are_within_the_bound(spread):
    s = pc.Step([700], [2], 1, 4, 128, 64, 16, F16, spread=spread)
    assert sharp.check(s, emulated(s)) <= 1.0


@pytest.mark.parametrize("case, first, last, times", [
    (([5000, 3, 0, 777], [1, 1, 1, 1], 4, 3, 128, 64, 128, F16), 1024, 1152, 0),
    (([2049] * 3, [1] * 3, 1, 16, 64, 32, 16, F16), 320, 352, 0),
    (([2049] * 3, [1] * 3, 1, 16, 64, 32, 16, F16), 320, 352, 2),
    (([1000], [1], 8, 4, 128, 64, 64, F16), 960, 1000, 0), (([1000], [1], 8, 4, 128, 64, 64, F16), 999, 1000, 0),
    (([20000], [1], 1, 8, 128, 64, 64, F16), 4000, 6000, 0), (([20000], [1], 1, 8, 128, 64, 64, F16), 4000, 5000, 2),
    (([6000], [1], 1, 8, 128, 64, 128, F32), 32, 33, 0),
    (([333, 100], [150, 17], 1, 3, 64, 64, 16, F16), 128, 192, 0),
])
def test_a_lost_run_is_not(case, first, last, times):
    s = pc.Step(*case, seed=5)
    assert sharp.worst(s, sharp.without(s, 0, first, last, times)) > 1.0


@pytest.mark.parametrize("ctx, new, dtype", [([20000, 40], [1, 1], F16), ([3001, 40], [7, 1], F16), ([900, 33], [60, 1], F16),
                                             ([5000, 40], [3, 1], F32)])
@pytest.mark.parametrize("at", [0.0, 0.37, 1.0])
def test_a_marked_block_shows(ctx, new, dtype, at):
    """Lost, doubled, or its last position lost: in steps of any length."""
    s = pc.Step(ctx, new, 2, 2, 128, 64, 16, dtype, packed=False)
    block = int(at * (pc.cdiv(ctx[0], 16) - 1))
    sharp.mark(s, [[block, block], [0, 1]])
    assert sharp.check(s, emulated(s)) <= 1.0
    first, last = 16 * block, min(16 * block + 16, ctx[0])
    for a, times in ((first, 0), (first, 2), (last - 1, 0)):
        assert sharp.worst(s, sharp.without(s, 0, a, last, times)) > 1.0


def test_a_lost_part_of_a_join_shows():
    """A CTA's part left out of the join, and one joined with the wrong weight."""
    s = pc.Step([40000], [1], 1, 8, 128, 64, 64, F16, seed=5)
    part = 40000 // 18
    assert sharp.worst(s, sharp.without(s, 0, 7 * part, 8 * part)) > 1.0
    assert sharp.worst(s, sharp.without(s, 0, 7 * part, 8 * part, 3)) > 1.0


def test_values_beside_an_outlier_are_judged():
    """One position with a scale 2^13 times the others' whose codes stand for
    (nearly) zero in every second dim: there the other positions' values count."""
    s = pc.Step([600], [1], 1, 4, 128, 64, 16, F16)
    sharp.outlier(s, 0, 0, 323)
    want = sharp.reference(s)[0]
    assert sharp.check(s, emulated(s)) <= 1.0
    lost = want.clone()
    s2 = pc.Step([600], [1], 1, 4, 128, 64, 16, F16)
    sharp.outlier(s2, 0, 0, 323)
    keep = s2.pools[4][s2.tables[0, 20], 0, 3].clone(), s2.pools[5][s2.tables[0, 20], 0, 3].clone()
    s2.pools[4].zero_(), s2.pools[5].zero_()
    s2.pools[4][s2.tables[0, 20], 0, 3], s2.pools[5][s2.tables[0, 20], 0, 3] = keep
    lost = sharp.reference(s2)[0].to(F16)
    assert sharp.worst(s, lost) > 1.0
