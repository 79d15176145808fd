"""``Qwen3Model.paged_step``'s host side with the kernels' calls replaced; CPU only."""

import types

import pytest
import torch

from torch2iron_amd import model as gm
from torch2iron_amd import ops

CFG = gm.Qwen3Config(n_layers=2, hidden=128, n_heads=1, n_kv_heads=1, vocab=32, intermediate=128)
CAP = 64


class _Step:
    """A model whose passes over the rows are counted, and whose verification says what the test wants."""

    def __init__(self, monkeypatch):
        self.passes, self.counts, self.next = 0, None, None
        real = ops._check_dev

        def check(name, t, dtype=None):
            if not isinstance(t, torch.Tensor) or (dtype is not None and t.dtype != dtype) or not t.is_contiguous():
                real(name, t, dtype)
                raise ValueError(name)

        def verify(logits, *args, **kw):
            return self.counts, self.next, torch.zeros(logits.shape[0])

        monkeypatch.setattr(ops, "_check_dev", check)
        monkeypatch.setattr(ops, "PagedPlan", lambda *a: None)
        monkeypatch.setattr(ops, "AdapterPlan", lambda *a: None)
        monkeypatch.setattr(ops, "rmsnorm", lambda x, *a, out=None, **kw: out)
        monkeypatch.setattr(ops, "lm_head_argmax", lambda *a, **kw: None)
        monkeypatch.setattr(ops, "verify_drafts", verify)
        self.model = types.SimpleNamespace(cfg=CFG, device=torch.device("cpu"), rope=torch.zeros(CAP, CFG.head_dim), norm=None,
                                           lm_head=None, layers=[None] * CFG.n_layers, _rows_pass=self._pass,
                                           micro=[types.SimpleNamespace(buf=types.SimpleNamespace(workspace=None))])

    def _pass(self, tokens, prep, attend, **kw):
        self.passes += 1
        return torch.zeros(tokens.numel(), CFG.hidden)

    def __call__(self, cache, batch, *args, **kw):
        return gm.Qwen3Model.paged_step(self.model, cache, batch, *args, **kw)


@pytest.fixture
def step(monkeypatch):
    return _Step(monkeypatch)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_lens_move_on_where_a_next_token_came_out(step):
    """A sequence whose next token is -1 (no room, no distribution) stays where it was, whatever its count says."""
    cache = gm.PagedCache(CFG, 4, 9, 4, "cpu", page_slots=16)
    cache.lens.copy_(_i32(5, 16, 40, 7))
    batch = gm.PagedBatch([3, 1, 4, 0], [1, 0, 3, 0], device="cpu")
    step.counts, step.next = _i32(1, 0, 2, 0), _i32(9, -1, -1, -1)
    got = step(cache, batch, torch.zeros(8, dtype=torch.int32))
    assert cache.lens.tolist() == [5 + 2 + 1, 16, 40, 7]
    assert got.counts.tolist() == [1, 0, 2, 0] and got.next_tokens.tolist() == [9, -1, -1, -1]
    step.counts, step.next = _i32(0, 0, 3, 0), _i32(0, 31, 2, -1)
    step(cache, batch, torch.zeros(8, dtype=torch.int32))
    assert cache.lens.tolist() == [8 + 2, 17, 44, 7]


def test_shapes_that_are_refused_before_the_pass(step):
    """tokens and adapter_ids are indexed by row and by sequence: as many values in another shape would be looked up out
    of range, behind the pages' writes."""
    cache = gm.PagedCache(CFG, 2, 9, 4, "cpu", page_slots=16)
    batch, tokens = gm.PagedBatch([2, 3], [0, 1], device="cpu"), torch.zeros(5, dtype=torch.int32)
    none = [gm.LayerAdapters()] * CFG.n_layers
    step.counts, step.next = _i32(0, 0), _i32(1, 1)
    step(cache, batch, tokens, adapters=none, adapter_ids=_i32(0, 0))
    assert step.passes == 1
    for kw in (dict(tokens=tokens.view(1, 5)), dict(tokens=tokens.view(5, 1)), dict(tokens=tokens[:4]), dict(tokens=tokens.view(1, 5, 1)),
               dict(adapters=none, adapter_ids=_i32(0, 0).view(1, 2)), dict(adapters=none, adapter_ids=_i32(0, 0).view(2, 1)),
               dict(adapters=none, adapter_ids=_i32(0))):
        with pytest.raises(ValueError, match="must hold|must be"):
            step(cache, batch, **{**dict(tokens=tokens), **kw})
    assert step.passes == 1


def test_adapters_that_are_no_layer_adapters_are_refused_before_the_pass(step):
    """A plain tuple has no projections by name, which came out in the layer that it was for, behind the writes of the others."""
    cache = gm.PagedCache(CFG, 2, 9, 4, "cpu", page_slots=16)
    batch, tokens = gm.PagedBatch([2, 3], device="cpu"), torch.zeros(5, dtype=torch.int32)
    step.counts, step.next = _i32(0, 0), _i32(1, 1)
    none = gm.LayerAdapters()
    for bad in ([none, tuple(none)], [none, None], [none, none._replace(o=torch.zeros(1))], [none, none._replace(o="o")]):
        with pytest.raises(ValueError, match="adapters"):
            step(cache, batch, tokens, adapters=bad, adapter_ids=_i32(0, 0))
    assert step.passes == 0
