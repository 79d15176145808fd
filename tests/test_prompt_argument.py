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


def _prompts(lengths, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2048, (n,), generator=g) for n in lengths]


@pytest.mark.gpu
def test_longer_ragged_prompts_keep_the_captured_steps(small):
    """The decode graphs do not depend on a packed prompt pass: another longest prompt captures nothing anew, and the
    calls before and behind it still replay what they captured."""
    small.generate(_prompts([5, 9, 2], 1), 10)
    step = small.micro[0].graphs["step"]
    for seed, lengths in enumerate(([5, 30, 2], [70, 1, 12], [3, 4, 5])):
        p = _prompts(lengths, seed)
        got = small.generate(p, 10)
        assert small.micro[0].graphs["step"] is step
        assert torch.equal(got, small.generate(p, 10, use_graph=False))
    batch = torch.stack(_prompts([20, 20, 20], 7))
    for mode in ("decode", "prefill"):
        want = small.generate(batch, 10, use_graph=False, prompt_mode=mode)
        assert torch.equal(small.generate(batch, 10, prompt_mode=mode), want)
        step = small.micro[0].graphs["step"]
        small.generate(_prompts([8, 64, 2], 8), 10)
        assert torch.equal(small.generate(batch, 10, prompt_mode=mode), want)
        assert small.micro[0].graphs["step"] is step
    assert torch.equal(small.generate(batch.tolist(), 10), small.generate(batch, 10))


@pytest.mark.gpu
def test_generate_refuses_what_is_no_integer(small):
    for bad in ([[1.9, 2.2], [3.7, 4.0], [1.0, 1.0]], torch.full((3, 2), 1.5)):
        with pytest.raises(ValueError):
            small.generate(bad, 2)
