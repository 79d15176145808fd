"""What the adapters' entry points refuse on the host, before anything is launched; CPU only."""

import ctypes

import pytest

from torch2iron_amd import _lib

FAKE = 0x10000          # an aligned, never-dereferenced address


def _plan(ids=FAKE, m=9, n=3, plan=FAKE, words=10**9):
    return _lib.load().t2i_adapter_plan(ids, m, n, plan, words, None)


def _add(y=FAKE, x=FAKE, m=9, k=128, n=128, plan=FAKE, words=10**9, a=FAKE, b=FAKE, scales=FAKE, pool=3, rank=8, parts=1, widths=None,
         paired=0, swiglu=0, out=2 * FAKE, ws=FAKE, nbytes=1 << 40):
    w = None if widths is None else (ctypes.c_int32 * len(widths))(*widths)
    return _lib.load().t2i_adapter_add(y, x, m, k, n, plan, words, a, b, scales, pool, rank, parts, w, paired, swiglu, out, ws, nbytes, None)


@pytest.mark.parametrize("kw", [dict(m=0), dict(m=1 << 24), dict(pool=0), dict(pool=512), dict(k=0), dict(k=48), dict(n=8), dict(n=24),
                                dict(k=1 << 21), dict(n=1 << 21), dict(rank=0), dict(rank=257), dict(parts=0), dict(parts=5),
                                dict(parts=1, paired=1), dict(parts=3, paired=1), dict(parts=2, n=256, widths=[128, 64]),
                                dict(parts=2, n=256, widths=[64, 192]), dict(parts=2, n=256, widths=[128, 256]),
                                dict(parts=2, n=256, widths=[-128, 384]),
                                dict(m=(1 << 24) - 1, n=1 << 20)], ids=str)
def test_sizes(kw):
    assert _add(**kw) == _lib.T2I_ERR_SHAPE


def test_pointers_and_values():
    E, lib = _lib, _lib.load()
    for name in ("y", "x", "plan", "a", "b", "out"):
        assert _add(**{name: None}) == E.T2I_ERR_NULL, name
        assert _add(**{name: 0x10008}) == E.T2I_ERR_ALIGN, name
    assert _add(scales=0x10002) == E.T2I_ERR_ALIGN and _add(ws=0x10008) == E.T2I_ERR_ALIGN
    assert _add(parts=2) == E.T2I_ERR_NULL
    assert _add(swiglu=1) == E.T2I_ERR_VALUE and _add(swiglu=1, paired=1, parts=2, out=FAKE) == E.T2I_ERR_VALUE
    need, words = lib.t2i_adapter_add_workspace_bytes(9, 3, 1, 8), lib.t2i_adapter_plan_words(9, 3)
    assert need > 9 * 16 * 4 and words > 9
    assert _add(nbytes=need - 1) == E.T2I_ERR_WORKSPACE and _add(ws=None) == E.T2I_ERR_WORKSPACE
    assert _add(words=words - 1) == E.T2I_ERR_WORKSPACE and _plan(words=words - 1) == E.T2I_ERR_WORKSPACE
    assert lib.t2i_adapter_add_workspace_bytes(9, 3, 5, 8) == 0 and lib.t2i_adapter_add_workspace_bytes(9, 3, 1, 257) == 0
    assert lib.t2i_adapter_add_workspace_bytes(0, 3, 1, 8) == 0 and lib.t2i_adapter_add_workspace_bytes(9, 512, 1, 8) == 0
    assert _plan(ids=None) == E.T2I_ERR_NULL and _plan(plan=None) == E.T2I_ERR_NULL
    assert _plan(ids=0x10002) == E.T2I_ERR_ALIGN and _plan(plan=0x10004) == E.T2I_ERR_ALIGN
    assert _plan(m=0) == E.T2I_ERR_SHAPE and _plan(n=0) == E.T2I_ERR_SHAPE and _plan(n=512) == E.T2I_ERR_SHAPE
    assert lib.t2i_adapter_plan_words(0, 3) == 0 and lib.t2i_adapter_plan_words(9, 512) == 0


@pytest.mark.parametrize("swiglu", [0, 1])
def test_out_over_a_part_of_y(swiglu):
    """Other rows than a workgroup's own would be written before they are read."""
    size = 9 * 128 * 2
    for y, out in ((FAKE, FAKE + 16), (FAKE, FAKE + size - 16), (FAKE + 16, FAKE), (FAKE + (size >> swiglu) - 16, FAKE)):
        assert _add(y=y, out=out, swiglu=swiglu, paired=swiglu, parts=1 + swiglu) == _lib.T2I_ERR_VALUE
