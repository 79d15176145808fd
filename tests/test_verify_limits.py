"""What the verification's entry point refuses on the host, before anything is launched; CPU only."""

import pytest

from torch2iron_amd import _lib

FAKE = 0x10000          # an aligned, never-dereferenced address


def _call(logits=FAKE, kind=0, stride=40, m=5, v=40, starts=FAKE, n=2, tokens=FAKE, u=FAKE, probs=FAKE, probs_stride=40, temps=FAKE,
          counts=FAKE, nxt=FAKE, lp=FAKE, ws=FAKE, nbytes=1 << 40):
    return _lib.load().t2i_verify_drafts(logits, kind, stride, m, v, starts, n, tokens, u, probs, probs_stride, temps, counts, nxt, lp,
                                         ws, nbytes, None)


@pytest.mark.parametrize("kw", [dict(m=0), dict(v=0), dict(n=0), dict(m=-1), dict(stride=39), dict(probs_stride=39),
                                dict(m=2**24, v=4096, stride=4096, probs_stride=4096), dict(n=2**16 + 1)], ids=str)
def test_sizes(kw):
    assert _call(**kw) == _lib.T2I_ERR_SHAPE


def test_pointers_and_values():
    E = _lib
    names = ("logits", "starts", "tokens", "u", "counts", "nxt", "lp")
    for name in names:
        assert _call(**{name: None}) == E.T2I_ERR_NULL, name
    for name in names + ("probs", "temps"):
        assert _call(**{name: 0x10002}) == E.T2I_ERR_ALIGN, name
    assert _call(logits=0x10001, kind=1) == E.T2I_ERR_ALIGN
    assert _call(kind=3) == E.T2I_ERR_VALUE and _call(kind=-1) == E.T2I_ERR_VALUE
    lib = _lib.load()
    for probs in (None, FAKE):
        need = lib.t2i_verify_drafts_workspace_bytes(5, 40, 2, probs is not None)
        assert need > 0
        assert _call(probs=probs, nbytes=need - 1) == E.T2I_ERR_WORKSPACE and _call(probs=probs, ws=None) == E.T2I_ERR_WORKSPACE
    assert _call(ws=0x10008) == E.T2I_ERR_ALIGN
    assert lib.t2i_verify_drafts_workspace_bytes(0, 40, 2, 0) == 0 and lib.t2i_verify_drafts_workspace_bytes(5, 40, 0, 0) == 0
