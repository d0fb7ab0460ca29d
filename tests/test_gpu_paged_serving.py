"""The serving classes over the paged cache, on the device: generation of
requests of different lengths, captured steps, ended and admitted requests."""

from __future__ import annotations

import json

import pytest
import torch

from kernelverify_b200 import decode_loop as dl

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(native_module):
    return dl.Decoder(dl.TINY)


@pytest.fixture(scope="module")
def native_module():
    from kernelverify_b200 import _native
    return _native.lib()


def prompts(model, lengths, seed=0):
    return [dl.make_prompt(model, 1, n, seed + i)[0].tolist() if n else [] for i, n in enumerate(lengths)]


def held(d):
    """Every page is held by one request or free."""
    lens, free = d.seqs.lens.tolist(), int(d.seqs.n_free.item())
    size = d.seqs.page_size
    used = [p for row, n in zip(d.seqs.block_tables.tolist(), lens) for p in row[:-(-n // size)]]
    assert sorted(used + d.seqs.free_pages[:free].tolist()) == list(range(d.seqs.pages))
    return lens


@pytest.mark.parametrize("page_size", [16, 64])
def test_every_attention_agrees_with_the_stock_composition(model, page_size):
    d = dl.PagedDecode(model, 4, 200, page_size=page_size, shadow=True)
    d.prefill(prompts(model, [5, 130, 0, 64]))
    for _ in range(3):
        assert d.step().item() == 0
    assert d.shadow_gap <= 4e-3 * max(1.0, d.shadow_mag) and d.shadow_mag > 0
    assert held(d) == [8, 133, 0, 67]


def test_captured_steps_are_the_eager_steps(model):
    runs = []
    for captured in (False, True):
        d = dl.PagedDecode(model, 3, 120)
        d.prefill(prompts(model, [33, 7, 64]))
        toks = [d.tok.clone()]
        if captured:
            d.capture()
        for _ in range(20):
            d.replay() if captured else d.step()
            toks.append(d.tok.clone())
        assert held(d) == [53, 27, 84]
        runs.append(torch.stack(toks))
        d.graph = None
    assert torch.equal(*runs)


def test_requests_end_and_others_take_their_pages(model):
    d = dl.PagedDecode(model, 3, 100, pages=9, page_size=16, shadow=True)
    d.prefill(prompts(model, [40, 20, 30]))
    d.step()
    d.release([0])
    assert held(d) == [0, 21, 31]
    d.step()
    assert held(d) == [0, 22, 32]
    d.prefill(prompts(model, [60, 0, 0], seed=5))        # into the row that was freed
    d.step()
    assert held(d) == [61, 23, 33]
    assert d.shadow_gap <= 4e-3 * max(1.0, d.shadow_mag)
    d.release([0, 1, 2])
    assert held(d) == [0, 0, 0] and int(d.seqs.n_free.item()) == 9


def test_shadow_steps_are_not_captured(model):
    d = dl.PagedDecode(model, 1, 64, page_size=16, shadow=True)
    d.prefill(prompts(model, [5]))
    with pytest.raises(ValueError, match="shadow"):
        d.capture()
    assert d.graph is None and held(d) == [5]


def test_a_step_that_does_not_fit_changes_nothing(model):
    d = dl.PagedDecode(model, 2, 64, pages=4, page_size=16)
    with pytest.raises(ValueError, match="fit"):
        d.prefill(prompts(model, [60, 17]))
    d.prefill(prompts(model, [32, 32]))
    before = d.tok.clone()
    assert d.step().item() == 1
    assert held(d) == [32, 32] and torch.equal(d.tok, before)


def test_the_command(model, capsys, monkeypatch):
    monkeypatch.setattr(dl, "QWEN3_4B", dl.TINY)
    assert dl.main(["--paged", "--tiny", "--prompt", "20", "70", "--batch", "3", "--steps", "5"]) == 0
    row = json.loads(capsys.readouterr().out)
    assert row["lens"] == [25, 75, 25] and row["ok"] and row["tps"] > 0
