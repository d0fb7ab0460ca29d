"""The host's part of generation over the paged cache, on the CPU: its
operators in plain form, every index checked before a tensor is touched."""

from __future__ import annotations

import pytest
import torch

from kernelverify_b200 import decode_loop as dl
from tests import paged_cpu


@pytest.fixture(scope="module")
def model():
    return dl.Decoder(dl.TINY, device="cpu", dtype=torch.float32)


@pytest.fixture
def decode(model, monkeypatch):
    paged_cpu.install(monkeypatch)

    def make(batch=3, max_len=64, **kw):
        return dl.PagedDecode(model, batch, max_len, page_size=16, **kw)
    return make


def prompts(model, lengths):
    return [dl.make_prompt(model, 1, n, i)[0].tolist() if n else [] for i, n in enumerate(lengths)]


def state(d):
    s = d.seqs
    return [x.clone() for x in (d.tok, d.live, s.lens, s.n_free, s.free_pages, s.block_tables)]


def test_generation_runs(decode, model):
    d = decode(shadow=True)
    d.prefill(prompts(model, [5, 0, 20]))
    for _ in range(2):
        assert d.step().item() == 0
    assert d.seqs.lens.tolist() == [7, 0, 22]
    assert 0 < d.shadow_gap <= 1e-4 * d.shadow_mag


@pytest.mark.parametrize("rows", [[3], [0, 7], [-4], [2 ** 40], [True, False, False], [1.0], ["0"]])
def test_release_checks_its_rows(decode, model, rows):
    """On a device a row outside the batch would be an assertion of the index
    kernel, which ends the process's context."""
    d = decode()
    d.prefill(prompts(model, [5, 9, 20]))
    before = state(d)
    with pytest.raises((ValueError, TypeError), match="row"):
        d.release(rows)
    assert all(torch.equal(x, y) for x, y in zip(before, state(d)))


@pytest.mark.parametrize("rows, lens", [([], [5, 9, 20]), ([0, 2, 0], [0, 9, 0]), ([-1], [5, 9, 0]),
                                        (range(3), [0, 0, 0]), (torch.tensor([1]), [5, 0, 20])])
def test_release_ends_requests(decode, model, rows, lens):
    d = decode()
    d.prefill(prompts(model, [5, 9, 20]))
    d.release(rows)
    assert d.seqs.lens.tolist() == lens and d.live.tolist() == [int(n > 0) for n in lens]
    assert d.seqs.n_free.item() == d.seqs.pages - sum(-(-n // 16) for n in lens)


@pytest.mark.parametrize("row, length", [(0, 65), (0, 2 ** 31), (3, 5), (-4, 5), (0, -1), (True, 5), (0, 5.0)])
def test_read_back_checks_row_and_length(decode, model, row, length):
    """A length past the row's table is not an index of the table."""
    d = decode()
    d.prefill(prompts(model, [5, 9, 20]))
    with pytest.raises((ValueError, TypeError), match="row|length"):
        d.caches[0].dequantized(row, length)


def test_read_back_to_the_end_of_a_row(decode, model):
    d = decode()
    d.prefill(prompts(model, [64, 9, 20]))
    k, v = d.caches[1].dequantized(0, 64)
    assert k.shape == v.shape == (64, 2, 64) and bool((k.abs().amax((1, 2)) > 0).all())
    assert torch.equal(d.caches[1].dequantized(-3, 10)[0], k[:10])
    assert d.caches[0].dequantized(2, 0)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("token", [1024, -1, 2 ** 40])
def test_prefill_checks_its_tokens(decode, model, token):
    """A token outside the vocabulary is not an index of the embedding."""
    d = decode()
    d.prefill(prompts(model, [5, 0, 20]))
    before = state(d)
    with pytest.raises(ValueError, match="token"):
        d.prefill([[], [3, token, 4], [1]])
    assert all(torch.equal(x, y) for x, y in zip(before, state(d)))
    d.prefill([[], [0, 1023], torch.tensor([5, 6])])
    assert d.seqs.lens.tolist() == [5, 2, 22]


def test_compared_steps_that_decode_nothing(decode, model):
    """With every attention compared: a step that does not fit, and one without
    a live row, return their status and change nothing."""
    d = decode(batch=2, pages=4, shadow=True)
    d.prefill(prompts(model, [32, 32]))
    before = state(d)
    assert d.step().item() == 1
    assert all(torch.equal(x, y) for x, y in zip(before, state(d)))
    d.release([0, 1])
    assert d.step().item() == 0
    assert d.seqs.lens.tolist() == [0, 0] and d.seqs.n_free.item() == 4


@pytest.mark.parametrize("lengths", [[], ["0", "5"], ["-3"]])
def test_the_command_checks_its_prompts(monkeypatch, capsys, lengths):
    monkeypatch.setattr(dl, "Decoder", None)                 # refused before a model is made
    with pytest.raises(SystemExit):
        dl.main(["--paged", "--tiny", "--prompt", *lengths])
    assert "--prompt" in capsys.readouterr().err
