"""What ``generate`` takes for prompts: one rule for lists of equal and of different lengths."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from torch2iron_amd import model as gm


def _model(batch=2, cap=8, vocab=16):
    m = SimpleNamespace(batch=batch, ctx_cap=cap, cfg=SimpleNamespace(vocab=vocab))
    m._prompt_list = lambda p: gm.Qwen3Model._prompt_list(m, p)
    return m


def _take(prompt, mode="prefill", **kw):
    return gm.Qwen3Model._prompt_argument(_model(**kw), prompt, mode)


@pytest.mark.parametrize("mode", ["prefill", "decode"])
@pytest.mark.parametrize("bad", [
    [[1.9, 2.2], [3.7, 4.0]], [[1.0, 2.0], [3.0, 4.0]], [[True, False], [True, True]], [[1, 2], torch.tensor([1.5, 2.0])],
    [[1, 2], [3, 16]], [[1, 2], [3, -1]], [[1, 2]], [[1], [2], [3]], [], [1, 2], [[], []],
    torch.tensor([[1.0, 2.0], [3.0, 4.5]]), torch.tensor([[1.0, 2.0], [3.0, float("nan")]]), np.array([[0.5, 1.0], [1.0, 1.0]])])
def test_refused(bad, mode):
    with pytest.raises(ValueError):
        _take(bad, mode)


def test_one_rule_for_any_lengths():
    """Lists, tensors and arrays mix, whether their lengths differ or not; equal ones make a batch."""
    for mode in ("prefill", "decode"):
        prompt, rows = _take([torch.tensor([1, 2]), [3, 4]], mode)
        assert rows is None and prompt.tolist() == [[1, 2], [3, 4]]
    prompt, rows = _take((np.array([1, 2]), torch.tensor([3], dtype=torch.int32)))
    assert prompt is None and [r.tolist() for r in rows] == [[1, 2], [3]]
    with pytest.raises(ValueError):
        _take([[1, 2], [3]], "decode")


def test_batches_of_whole_numbers_pass_as_they_are():
    for p in (torch.tensor([[1, 2], [3, 4]]), torch.tensor([[1, 2], [3, 4]], dtype=torch.uint8), np.array([[1, 2], [3, 4]]),
              torch.tensor([[1.0, 2.0], [3.0, 4.0]])):
        prompt, rows = _take(p)
        assert rows is None and prompt.to(torch.int32).tolist() == [[1, 2], [3, 4]]


@pytest.fixture(scope="module")
def small(gpu):
    cfg = gm.Qwen3Config(n_layers=2, vocab=2048)
    return gm.Qwen3Model(gm.random_qwen3_tensors(cfg, seed=62, weights="centered"), cfg, batch=3, ctx_cap=96, device=gpu)


@pytest.mark.gpu
def test_generate_refuses_what_is_no_integer(small):
    for bad in ([[1.9, 2.2], [3.7, 4.0], [1.0, 1.0]], torch.full((3, 2), 1.5)):
        with pytest.raises(ValueError):
            small.generate(bad, 2)
