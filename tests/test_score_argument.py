"""``score`` refuses a number of alternatives that it cannot give before it touches the cache; CPU only."""

from types import SimpleNamespace

import pytest

from torch2iron_amd import ops
from torch2iron_amd.model import Qwen3Model


@pytest.mark.parametrize("top_k,vocab", [(-1, 2048), (ops.MAX_TOP_K + 1, 2048), (9, 8)])
def test_top_k(top_k, vocab):
    def packed_pass(prompts):
        raise AssertionError("the cache was overwritten")

    m = SimpleNamespace(cfg=SimpleNamespace(vocab=vocab), _prompt_list=lambda p: p, _packed_pass=packed_pass)
    with pytest.raises(ValueError, match="top_k"):
        Qwen3Model.score(m, [[1, 2]], top_k=top_k)
