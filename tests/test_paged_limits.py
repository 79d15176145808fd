"""What the paged entry points refuse on the host, before anything is launched; CPU only."""

import pytest

from torch2iron_amd import _lib

FAKE = 0x10000          # an aligned, never-dereferenced address
ODD = 0x10002


def _plan(starts=FAKE, ctx=FAKE, n=2, rows=9, max_pages=4, page=16, hq=16, hkv=8, plan=FAKE, words=None):
    lib = _lib.load()
    words = lib.t2i_paged_plan_words(rows, n, hq, hkv) if words is None else words
    return lib.t2i_paged_plan(starts, ctx, n, rows, max_pages, page, hq, hkv, plan, words, None)


def _prep(qkv=FAKE, rows=9, plan=FAKE, words=10**6, pages=FAKE, n=2, max_pages=4, n_pages=7, page=16, hq=16, hkv=8, d=128,
          qn=FAKE, eps=1e-6, rope=FAKE, style=0, q=FAKE, k=FAKE, v=FAKE):
    return _lib.load().t2i_paged_qk_rope_kv(qkv, rows, plan, words, pages, n, max_pages, n_pages, page, hq, hkv, d, qn, qn, eps,
                                            rope, style, q, k, v, None)


def _attn(q=FAKE, rows=9, plan=FAKE, words=10**6, pages=FAKE, n=2, max_pages=4, n_pages=7, page=16, hq=16, hkv=8, d=128, k=FAKE,
          v=FAKE, out=FAKE, sums=None, ws=FAKE, nbytes=1 << 30):
    return _lib.load().t2i_paged_attention(q, rows, plan, words, pages, n, max_pages, n_pages, page, hq, hkv, d, k, v, out, sums, ws,
                                           nbytes, None)


SIZES = [dict(n=0), dict(n=4097), dict(rows=0), dict(rows=-3), dict(rows=1 << 24), dict(max_pages=0), dict(page=0), dict(page=8),
         dict(page=24), dict(page=131072), dict(max_pages=1 << 20), dict(hq=0), dict(hq=15), dict(hkv=0), dict(hkv=17), dict(hq=2048)]


@pytest.mark.parametrize("call", [_plan, _prep, _attn])
@pytest.mark.parametrize("bad", SIZES, ids=str)
def test_sizes(call, bad):
    extra = dict(words=10**9) if call is _plan else {}
    assert call(**bad, **extra) == _lib.T2I_ERR_SHAPE
    assert _lib.load().t2i_last_error()


def test_too_many_tiles_for_32_bits():
    """Tiles times key blocks, in which the plan counts, stay below 2^31 / 32."""
    big = dict(rows=1 << 20, n=1, max_pages=8192, page=1024, hq=64, hkv=1, words=10**9)
    assert _plan(**big) == _lib.T2I_ERR_SHAPE


@pytest.mark.parametrize("call,names", [(_plan, ("starts", "ctx", "plan")), (_prep, ("qkv", "plan", "pages", "qn", "rope", "q", "k", "v")),
                                        (_attn, ("q", "plan", "pages", "k", "v", "out"))])
def test_null_and_misaligned_pointers(call, names):
    for name in names:
        assert call(**{name: None}) == _lib.T2I_ERR_NULL, name
        assert call(**{name: 0x10001}) == _lib.T2I_ERR_ALIGN, name
    for name in set(names) & {"qkv", "qn", "rope", "q", "k", "v", "out"}:
        assert call(**{name: ODD}) == _lib.T2I_ERR_ALIGN, name


def test_other_arguments():
    E = _lib
    lib = _lib.load()
    words, nbytes = lib.t2i_paged_plan_words(9, 2, 16, 8), lib.t2i_paged_attention_workspace_bytes(9, 16, 8)
    assert words > 0 and nbytes > 0
    assert _plan(words=words - 1) == E.T2I_ERR_WORKSPACE
    assert _prep(words=words - 1) == E.T2I_ERR_WORKSPACE and _attn(words=words - 1) == E.T2I_ERR_WORKSPACE
    assert _attn(nbytes=nbytes - 1) == E.T2I_ERR_WORKSPACE and _attn(ws=None) == E.T2I_ERR_WORKSPACE
    assert _attn(ws=0x10008) == E.T2I_ERR_ALIGN and _attn(sums=ODD) == E.T2I_ERR_ALIGN
    assert _prep(d=64) == E.T2I_ERR_SHAPE and _attn(d=256) == E.T2I_ERR_SHAPE
    assert _prep(n_pages=0) == E.T2I_ERR_SHAPE and _attn(n_pages=-1) == E.T2I_ERR_SHAPE
    assert _prep(style=2) == E.T2I_ERR_VALUE and _prep(eps=0.0) == E.T2I_ERR_VALUE and _prep(eps=float("nan")) == E.T2I_ERR_VALUE
    assert lib.t2i_paged_plan_words(0, 2, 16, 8) == 0 and lib.t2i_paged_plan_words(9, 2, 16, 7) == 0
    assert lib.t2i_paged_attention_workspace_bytes(0, 16, 8) == 0 and lib.t2i_paged_attention_workspace_bytes(9, 16, 7) == 0
