"""Drafted trees of many sequences, several tiles and every row range of the linears: what one to five small trees
do not reach."""

import pytest
import torch
from test_gpu_ragged import _check, _commit_reference, _tree_case, _tree_reference
from test_gpu_ragged_model import CAP, _check_greedy, _prompts, setup  # noqa: F401 (a fixture)

from torch2iron_amd import model as gm
from torch2iron_amd import ops

pytestmark = pytest.mark.gpu


def _many(b, cap, n, seed):
    """Contexts and counts of b sequences: short and long ones, some without nodes, some outside the cache."""
    g = torch.Generator().manual_seed(seed)
    ctx = torch.randint(0, cap - n + 1, (b,), generator=g).tolist()
    counts = torch.randint(1, n + 1, (b,), generator=g).tolist()
    for i in range(0, b, 7):
        counts[i] = 0
    for i in range(3, b, 11):
        ctx[i] = (-1, cap, cap - counts[i] + 1)[i % 3]
    for i in range(5, b, 13):
        counts[i], ctx[i] = n, cap - n
    return ctx, counts


# more than 64 sequences: later windows of the scan, a window of empty ones, several tiles beside each other
@pytest.mark.parametrize("b,hq,hkv,cap,n,kind", [(65, 4, 2, 300, 8, "random"), (150, 4, 1, 200, 13, "random"),
                                                 (150, 8, 8, 90, 5, "chain"), (130, 16, 2, 150, 40, "random")])
def test_tree_attention_of_many_sequences(gpu, b, hq, hkv, cap, n, kind):
    ctx, counts = _many(b, cap, n, b + n)
    for first in (0, 1):
        if first:                              # nothing but empty sequences in the first window
            counts = [0 if i < 64 else c for i, c in enumerate(counts)]
        q, parents, ctx_t, counts_t, kc, vc, _ = _tree_case(gpu, hq, hkv, cap, ctx, n, counts, kind)
        ref, mag = _tree_reference(q, parents, ctx, counts, kc, vc, cap)
        out = torch.full((b * n, hq * 128), 7.0, dtype=q.dtype, device=gpu)
        got = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t, out=out).view(ref.shape)
        for i, c in enumerate(counts):
            _check(got[i, :c], ref[i, :c], mag[i, :c], f"sequence {i}")
            assert (got[i, c:] == 7.0).all()


@pytest.mark.parametrize("hq,hkv,n,ctx,counts", [
    (32, 4, 64, [100, 0, 37, 200, 64], [64, 1, 40, 32, 33]),          # two tiles of 256, one of them unused by some
    (64, 1, 64, [900, 5, 0], [64, 3, 20]),                            # sixteen tiles
    (16, 2, 40, [130, 260, 3], [40, 16, 17]), (10, 1, 64, [700, 0, 9, 50], [64, 0, 25, 26])])
def test_tree_attention_of_several_tiles(gpu, hq, hkv, n, ctx, counts):
    """Sequences with fewer nodes than the widest leave whole tiles out."""
    cap = 1000
    q, parents, ctx_t, counts_t, kc, vc, _ = _tree_case(gpu, hq, hkv, cap, ctx, n, counts, "random")
    ref, mag = _tree_reference(q, parents, ctx, counts, kc, vc, cap)
    out = torch.full((len(ctx) * n, hq * 128), 7.0, dtype=q.dtype, device=gpu)
    got = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t, out=out).view(ref.shape)
    for i, c in enumerate(counts):
        _check(got[i, :c], ref[i, :c], mag[i, :c], f"sequence {i}")
        assert (got[i, c:] == 7.0).all()


def test_tree_commit_of_many_sequences(gpu):
    b, n, cap, layers, hkv = 150, 13, 200, 2, 2
    ctx, counts = _many(b, cap, n, 4)
    _, parents, ctx_t, counts_t, kc, vc, _ = _tree_case(gpu, 2, hkv, cap, ctx, n, counts, "random")
    kc, vc = (torch.stack([c.nan_to_num(3.0), c.nan_to_num(5.0) + 1]) for c in (kc, vc))
    g = torch.Generator().manual_seed(3)
    tokens, picks = (torch.randint(0, 2, (b, n), generator=g, dtype=torch.int32) for _ in range(2))
    ref = _commit_reference(tokens, parents.tolist(), picks, ctx, counts, kc, vc, cap)
    path, m, nxt, out = ops.tree_commit(tokens.to(gpu), parents, picks.to(gpu), ctx_t, kc, vc, node_counts=counts_t)
    assert path.cpu().tolist() == ref[0].tolist() and (m.tolist(), nxt.tolist(), out.tolist()) == ref[1:4]
    assert torch.equal(kc, ref[4]) and torch.equal(vc, ref[5]) and kc.shape[0] == layers


def _drafts(true, n, g):
    """A random tree of n nodes with the tokens to come along one of its paths, decoys elsewhere."""
    parents = [-1] + [int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(1, n)]
    tokens = torch.randint(0, 2048, (n,), generator=g, dtype=torch.int32)
    at, depth = 0, 0
    for i in range(1, n):
        if parents[i] == at and depth < len(true) and (i % 2 or n - i < 8):
            tokens[i], at, depth = true[depth], i, depth + 1
    return tokens, torch.tensor(parents, dtype=torch.int32)


@pytest.mark.parametrize("b,n", [(4, 26), (9, 64), (2, 32)], ids=["104_rows", "576_rows", "64_rows"])
def test_verify_tree_at_every_row_range(gpu, setup, b, n):  # noqa: F811
    """Up to 64 rows the norms run inside the linears, above on their own, and from 512 with row sums handed over
    (the tree attention gives none): all emit what greedy decode does."""
    cfg, t, o32, o16 = setup
    assert (b * n >= ops.PROMPT_GEMM_ROWS) == (b == 9)
    m = gm.Qwen3Model(t, cfg, batch=b, ctx_cap=CAP, device=gpu)
    prompts = _prompts(cfg, [1 + (37 * i) % 90 for i in range(b)], 11)
    true = m.generate(prompts, 40).tolist()
    m.history = None
    m.prefill_packed(prompts)
    out = [[int(x)] for x in m.tokens.tolist()]
    g = torch.Generator().manual_seed(12)
    accepted = 0
    for step in range(3):
        trees = [_drafts(true[i][len(out[i]):], n, g) for i in range(b)]
        counts = [n if (i + step) % 3 else max(1, n // 2 + i - step) for i in range(b)]
        counts[step % b] = 0 if step == 1 else counts[step % b]
        before = m.positions.tolist()
        got, k = m.verify_tree(torch.stack([a for a, _ in trees]).to(gpu), torch.stack([p for _, p in trees]).to(gpu),
                               node_counts=torch.tensor(counts, dtype=torch.int32, device=gpu))
        got, k = got.tolist(), k.tolist()
        for i in range(b):
            assert (k[i] == 0) == (counts[i] == 0) and got[i][k[i]:] == [-1] * (n - k[i])
            out[i] += got[i][:k[i]]
        assert m.positions.tolist() == [p + x for p, x in zip(before, k)] and m.tokens.tolist() == [o[-1] for o in out]
        accepted += sum(x - 1 for x in k if x)
    assert accepted >= 2 * b, f"{accepted} drafted tokens accepted"
    for _ in range(2):                         # plain decode goes on from the cache that the trees left
        m.forward_step()
        ops.greedy_advance(m.keys, m.tokens, m.positions, None, m.step)
        for o, x in zip(out, m.tokens.tolist()):
            o.append(x)
    for i, p in enumerate(prompts):
        _check_greedy(o32, o16, p, out[i], f"sequence {i}")


def test_verify_tree_leaves_the_token_record(gpu, setup):  # noqa: F811
    """``history`` and ``step``, the record of equal steps, stay: sequences accept different numbers."""
    cfg, t, _, _ = setup
    m = gm.Qwen3Model(t, cfg, batch=2, ctx_cap=CAP, device=gpu)
    prompts = _prompts(cfg, [5, 9], 13)
    m.generate(prompts, 4)
    m.prefill_packed(prompts)
    record = m.history.clone(), m.step.clone()
    tokens, parents = _drafts([], 6, torch.Generator().manual_seed(1))
    m.verify_tree(tokens.repeat(2, 1).to(gpu), parents.repeat(2, 1).to(gpu))
    assert torch.equal(m.history, record[0]) and torch.equal(m.step, record[1])
