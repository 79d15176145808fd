"""The packed plan (host code) and the refusals of the ragged entry points: CPU only, nothing is launched."""

import random

import pytest
import torch

from torch2iron_amd import _lib
from torch2iron_amd import ops

FAKE = 0x10000          # an aligned, never-dereferenced address
ODD = 0x10002
E = _lib
ROWS, KEYS = 128, 64


def _tables(plan):
    t, n = plan.table, plan.rows
    items = t[2 * n:2 * n + 8 * plan.n_items].view(-1, 8).tolist()
    at = 2 * n + 8 * plan.n_items
    end = at + 8 * plan.n_merges
    assert t.numel() == end + plan.n_bins + 1
    return t[:n].tolist(), t[n:2 * n].tolist(), items, t[at:end].view(-1, 8).tolist(), t[end:].tolist()


def _batches():
    rng = random.Random(3)
    yield [1], [0], None, 4, 2, 8
    yield [0, 0], [0, 5], None, 4, 2, 8
    yield [3], [8000], None, 8, 1, 8192
    yield [8001], [0], None, 32, 8, 8192
    yield [1] * 24 + [509, 701], [3000 + 40 * i for i in range(24)] + [2005, 3990], None, 32, 8, 4800
    for _ in range(60):
        n = rng.choice([1, 2, 5, 17])
        cap = rng.choice([64, 777, 5000, 20000])
        lengths = [rng.choice([0, 1, rng.randrange(0, min(cap, 900) + 1)]) for _ in range(n)]
        starts = [rng.randrange(0, cap - x + 1) for x in lengths]
        rows = rng.sample(range(n + 3), n) if rng.random() < 0.5 else None
        hkv = rng.choice([1, 2, 8])
        yield lengths, starts, rows, hkv * rng.choice([1, 2, 3, 8, 10]), hkv, cap


@pytest.mark.parametrize("lengths,starts,rows,hq,hkv,cap", list(_batches()))
def test_plan_covers_every_pair_once(lengths, starts, rows, hq, hkv, cap):
    """Every (row, head) pair and every key block it attends is in exactly one item, every item in one bin; cut
    tiles have one merge over their own parts; rows go to their slots; cut plans have even bins."""
    plan = ops.PackedPlan(lengths, hq, hkv, cap, "cpu", starts=starts, cache_rows=rows)
    pos, crow, items, merges, bins = _tables(plan)
    g, at, want = hq // hkv, 0, {}
    for s, (n, start) in enumerate(zip(lengths, starts)):
        c = s if rows is None else rows[s]
        assert pos[at:at + n] == list(range(start, start + n)) and crow[at:at + n] == [c] * n
        assert (plan.first_rows[s], plan.last_rows[s]) == (at, at + n - 1)
        for j0 in range(0, n * g, ROWS):
            last = (min(j0 + ROWS, n * g) - 1) // g
            want[(at, n, start, c, j0)] = (start + last) // KEYS + 1
        at += n
    assert plan.rows == at == sum(lengths)
    got, parts = {}, {}
    for row0, n, start, c, j0, k0, k1, part in items:
        assert k0 < k1
        got.setdefault((row0, n, start, c, j0), []).append((k0, k1, part))
    assert got.keys() == want.keys()
    for key, blocks in want.items():
        ranges = sorted(got[key])
        assert ranges[0][0] == 0 and ranges[-1][1] == blocks
        assert all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
        if len(ranges) == 1:
            assert ranges[0][2] == -1
        else:
            parts[(key[0], key[1], key[4])] = [p for _, _, p in ranges]
    joined = {}
    for row0, n, j0, first, count, e, *_ in merges:
        assert parts[row0, n, j0] == list(range(first, first + count))
        joined.setdefault((row0, n, j0), []).append(e)
    assert joined == {k: list(range(0, min(k[1] * g - k[2], ROWS), 8)) for k in parts}
    used = [i[7] for i in items if i[7] >= 0]
    assert sorted(used) == list(range(plan.n_parts))
    assert bins[0] == 0 and bins[-1] == len(items) and all(a < b for a, b in zip(bins, bins[1:]))
    if plan.n_parts:          # even shares: about one round of workgroups
        assert plan.n_bins * hkv <= 512 + hkv
        loads = [sum(i[6] - i[5] for i in items[a:b]) for a, b in zip(bins, bins[1:])]
        assert max(loads) <= 2 * (sum(loads) / len(loads)) + 3
    else:                     # a workgroup a tile
        assert bins == list(range(len(items) + 1))


def test_plan_splits_few_rows_over_a_long_context_only():
    assert ops.PackedPlan([3], 8, 1, 8192, "cpu", starts=[8000]).n_parts >= 4
    assert ops.PackedPlan([512] * 16, 16, 8, 640, "cpu").n_parts == 0
    assert ops.PackedPlan([1] * 4, 16, 8, 640, "cpu", starts=[100] * 4).n_parts == 0


@pytest.mark.parametrize("kw", [
    dict(lengths=[]), dict(lengths=[-1]), dict(lengths=[5], starts=[60]), dict(lengths=[5], starts=[-1]),
    dict(lengths=[1], starts=[2**31 - 1]), dict(lengths=[2**31]), dict(lengths=[1, 1], starts=[0]),
    dict(lengths=[1, 1], cache_rows=[1, 1]), dict(lengths=[1, 1], cache_rows=[0]), dict(lengths=[1, 1], cache_rows=[0, -1]),
    dict(lengths=[1, 1], cache_rows=[0, 5], n_cache_rows=4), dict(lengths=[1, 1], n_cache_rows=1),
    dict(lengths=[1], heads=(6, 4)), dict(lengths=[1], heads=(2, 4)), dict(lengths=[1], heads=(4, 0)), dict(lengths=[1], cap=0)])
def test_plan_refusals(kw):
    hq, hkv = kw.pop("heads", (16, 8))
    with pytest.raises(ValueError):
        ops.PackedPlan(kw.pop("lengths"), hq, hkv, kw.pop("cap", 64), "cpu", **kw)


def test_plan_entry_point_checks_its_table():
    lib = _lib.load()
    n = torch.tensor([300], dtype=torch.int32)
    s = torch.zeros(1, dtype=torch.int32)
    sizes = torch.zeros(6, dtype=torch.int64)
    call = (n.data_ptr(), s.data_ptr(), None, 1, 16, 8, 1, 512)
    assert lib.t2i_packed_plan(*call, None, 0, sizes.data_ptr()) == 0
    words = int(sizes[5])
    table = torch.full((words + 1,), -7, dtype=torch.int32)
    assert lib.t2i_packed_plan(*call, table.data_ptr(), words - 1, sizes.data_ptr()) == E.T2I_ERR_WORKSPACE
    assert (table == -7).all()
    assert lib.t2i_packed_plan(*call, table.data_ptr(), words, sizes.data_ptr()) == 0
    assert table[-1] == -7 and (table[:-1] != -7).all()
    assert lib.t2i_packed_plan(None, *call[1:], None, 0, sizes.data_ptr()) == E.T2I_ERR_NULL


def test_packed_entry_points_refuse():
    lib = _lib.load()

    def prep(qkv=FAKE, rows=5, pos=FAKE, cache=2, hq=16, hkv=8, d=128, eps=1e-6, style=0, q=FAKE, kc=FAKE, cap=64):
        return lib.t2i_packed_qk_rope_kv(qkv, rows, pos, FAKE, cache, hq, hkv, d, FAKE, FAKE, eps, FAKE, style, q, kc, FAKE, cap, None)

    for kw, code in ((dict(qkv=None), E.T2I_ERR_NULL), (dict(pos=None), E.T2I_ERR_NULL), (dict(q=ODD), E.T2I_ERR_ALIGN),
                     (dict(pos=ODD), E.T2I_ERR_ALIGN), (dict(rows=0), E.T2I_ERR_SHAPE), (dict(d=64), E.T2I_ERR_SHAPE),
                     (dict(hq=12), E.T2I_ERR_SHAPE), (dict(cache=0), E.T2I_ERR_SHAPE), (dict(cap=0), E.T2I_ERR_SHAPE),
                     (dict(eps=0.0), E.T2I_ERR_VALUE), (dict(style=2), E.T2I_ERR_VALUE), (dict(kc=ODD), E.T2I_ERR_ALIGN)):
        assert prep(**kw) == code, kw

    def attn(q=FAKE, rows=5, items=FAKE, n_items=3, merges=None, n_merges=0, parts=0, bins=FAKE, n_bins=3, hq=16, hkv=8, d=128, cache=2, cap=64,
             out=FAKE, sums=None, ws=None, nbytes=0):
        return lib.t2i_packed_attention(q, rows, items, n_items, merges, n_merges, parts, bins, n_bins, hq, hkv, d, FAKE, FAKE, cache, cap, out,
                                        sums, ws, nbytes, None)

    need = lib.t2i_packed_attention_workspace_bytes(2, 8)
    assert need > 0 and lib.t2i_packed_attention_workspace_bytes(0, 8) == 0
    split = dict(merges=FAKE, n_merges=1, parts=2)
    for kw, code in ((dict(q=None), E.T2I_ERR_NULL), (dict(out=ODD), E.T2I_ERR_ALIGN), (dict(items=ODD), E.T2I_ERR_ALIGN),
                     (dict(sums=ODD), E.T2I_ERR_ALIGN), (dict(rows=0), E.T2I_ERR_SHAPE), (dict(n_items=0), E.T2I_ERR_SHAPE),
                     (dict(parts=2), E.T2I_ERR_SHAPE), (dict(hq=15), E.T2I_ERR_SHAPE), (dict(hq=2048), E.T2I_ERR_SHAPE),
                     (dict(d=256), E.T2I_ERR_SHAPE), (dict(n_bins=2**29), E.T2I_ERR_SHAPE), (dict(n_bins=0), E.T2I_ERR_SHAPE),
                     (dict(bins=None), E.T2I_ERR_NULL), (dict(bins=ODD), E.T2I_ERR_ALIGN), (dict(cap=2**23 + 1), E.T2I_ERR_SHAPE), (split, E.T2I_ERR_WORKSPACE),
                     (dict(**split, ws=FAKE, nbytes=need - 1), E.T2I_ERR_WORKSPACE),
                     (dict(**split, ws=FAKE + 8, nbytes=need), E.T2I_ERR_ALIGN)):
        assert attn(**kw) == code, kw


def test_tree_entry_points_refuse():
    lib = _lib.load()

    def prep(parents=FAKE, ctx=FAKE, counts=None, b=2, n=8, hq=16, hkv=8, d=128, eps=1e-6, cap=64, q=FAKE):
        return lib.t2i_tree_qk_rope_kv(FAKE, parents, ctx, counts, b, n, hq, hkv, d, FAKE, FAKE, eps, FAKE, 0, q, FAKE, FAKE, cap, None)

    def attn(parents=FAKE, ctx=FAKE, counts=None, b=2, n=8, hq=16, hkv=8, d=128, cap=64, q=FAKE, ws=None, nbytes=0):
        return lib.t2i_tree_attention(q, parents, ctx, counts, b, n, hq, hkv, d, FAKE, FAKE, cap, FAKE, ws, nbytes, None)

    def commit(parents=FAKE, ctx=FAKE, counts=None, b=2, n=8, hq=16, hkv=8, d=128, cap=64, layers=3, tokens=FAKE, out=FAKE + 4096,
               kc=FAKE, path=FAKE):
        return lib.t2i_tree_commit(tokens, parents, FAKE, ctx, counts, layers, b, n, hkv, d, kc, FAKE, cap, path, FAKE, FAKE, out, None)

    shared = ((dict(parents=None), E.T2I_ERR_NULL), (dict(ctx=None), E.T2I_ERR_NULL), (dict(parents=ODD), E.T2I_ERR_ALIGN),
              (dict(counts=ODD), E.T2I_ERR_ALIGN), (dict(n=0), E.T2I_ERR_SHAPE), (dict(n=65), E.T2I_ERR_SHAPE),
              (dict(b=0), E.T2I_ERR_SHAPE), (dict(n=9, cap=8), E.T2I_ERR_SHAPE), (dict(d=64), E.T2I_ERR_SHAPE))
    for f in (prep, attn, commit):
        for kw, code in shared:
            assert f(**kw) == code, (f.__name__, kw)
    assert prep(eps=-1.0) == E.T2I_ERR_VALUE and prep(hq=17) == E.T2I_ERR_SHAPE and prep(q=ODD) == E.T2I_ERR_ALIGN
    assert attn(hq=17) == E.T2I_ERR_SHAPE and attn(q=None) == E.T2I_ERR_NULL and attn(q=ODD) == E.T2I_ERR_ALIGN
    need = lib.t2i_tree_attention_workspace_bytes(1, 8, 16, 8, 32768)
    assert need > 0
    assert attn(b=1, cap=32768) == E.T2I_ERR_WORKSPACE and attn(b=1, cap=32768, ws=FAKE, nbytes=need - 1) == E.T2I_ERR_WORKSPACE
    assert attn(b=1, cap=32768, ws=FAKE + 8, nbytes=need) == E.T2I_ERR_ALIGN
    assert lib.t2i_tree_attention_workspace_bytes(1, 65, 16, 8, 32768) == 0
    assert commit(layers=0) == E.T2I_ERR_SHAPE and commit(tokens=None) == E.T2I_ERR_NULL and commit(kc=ODD) == E.T2I_ERR_ALIGN
    assert commit(path=ODD) == E.T2I_ERR_ALIGN and commit(out=FAKE) == E.T2I_ERR_VALUE


def test_logprobs_entry_point_refuses():
    lib = _lib.load()

    def call(x=FAKE, kind=0, stride=5000, m=2, v=5000, tokens=FAKE, k=3, lp=FAKE, ent=FAKE, top=FAKE, ids=FAKE, ws=None, nbytes=0):
        return lib.t2i_token_logprobs(x, kind, stride, m, v, tokens, k, lp, ent, top, ids, ws, nbytes, None)

    need = lib.t2i_token_logprobs_workspace_bytes(2, 5000, 3)
    for kw, code in ((dict(x=None), E.T2I_ERR_NULL), (dict(lp=None), E.T2I_ERR_NULL), (dict(top=None), E.T2I_ERR_NULL),
                     (dict(kind=3), E.T2I_ERR_VALUE), (dict(kind=-1), E.T2I_ERR_VALUE), (dict(k=33), E.T2I_ERR_VALUE),
                     (dict(k=-1), E.T2I_ERR_VALUE), (dict(v=2, k=3), E.T2I_ERR_VALUE), (dict(stride=4999), E.T2I_ERR_SHAPE),
                     (dict(m=0), E.T2I_ERR_SHAPE), (dict(v=0), E.T2I_ERR_SHAPE), (dict(x=ODD), E.T2I_ERR_ALIGN),
                     (dict(x=FAKE + 1, kind=1), E.T2I_ERR_ALIGN), (dict(tokens=ODD), E.T2I_ERR_ALIGN), (dict(), E.T2I_ERR_WORKSPACE),
                     (dict(ws=FAKE, nbytes=need - 1), E.T2I_ERR_WORKSPACE), (dict(ws=FAKE + 8, nbytes=need), E.T2I_ERR_ALIGN)):
        assert call(**kw) == code, kw
    assert need > 0 and lib.t2i_token_logprobs_workspace_bytes(2, 5000, 33) == 0


def test_ops_refuse_host_tensors():
    bf, i32 = torch.bfloat16, torch.int32
    x, i = torch.zeros(4, 2, 128, dtype=bf), torch.zeros(2, 2, dtype=i32)
    c = torch.zeros(1, 1, 16, 128, dtype=bf)
    plan = ops.PackedPlan([4], 2, 1, 16, "cpu")
    for f in (lambda: ops.packed_attention(x, plan, c, c),
              lambda: ops.packed_qk_rope_kv(x, plan, x[0, 0], x[0, 0], 1e-6, x[0], c, c),
              lambda: ops.tree_attention(x, i, i[0], 1, c, c),
              lambda: ops.tree_qk_rope_kv(x, i, i[0], 2, 1, x[0, 0], x[0, 0], 1e-6, x[0], c, c),
              lambda: ops.tree_commit(i, i, i, i[0], c, c),
              lambda: ops.token_logprobs(x[0].float(), i[0])):
        with pytest.raises(ValueError, match="GPU tensor"):
            f()


@pytest.mark.parametrize("bad", [[1.5, 2.0], [True, False]], ids=["float", "bool"])
def test_prompts_that_are_no_integers_are_refused(bad):
    """They are not rounded to token ids; lists and tensors of integers pass."""
    from types import SimpleNamespace

    from torch2iron_amd.model import Qwen3Model
    m = SimpleNamespace(batch=2, ctx_cap=8, cfg=SimpleNamespace(vocab=16))
    for p in (bad, torch.tensor(bad)):
        with pytest.raises(ValueError, match="integers"):
            Qwen3Model._prompt_list(m, [[1, 2], p])
    got = Qwen3Model._prompt_list(m, [[1, 2], torch.tensor([3], dtype=torch.int64)])
    assert [p.tolist() for p in got] == [[1, 2], [3]] and all(p.dtype == torch.int32 for p in got)
