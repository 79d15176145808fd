"""Packed prompts and drafted trees on the MI355X against plain float64 attention.

Tolerance of the attention, elementwise: the softmax weights w_j enter P . V rounded to bf16 (each
off by at most 2^-8 relative) and are normalised by the sum of the rounded ones, so an output
sum w_j v_j / sum w_j moves by at most 2^-8 sum p_j |v_j - out| <= 2^-8 (sum p_j |v_j| + |out|);
its own rounding to bf16 adds 2^-8 |out|; second-order terms and fp32 scores, exponentials and
sums (scores of up to 40 with 128 terms: 128 * 2^-24 * 40 < 4e-4 relative of a weight at the
very worst, a tenth of that in the mean over keys) are covered by 2^-8 more of |out| and 2e-4 of the
largest sum p_j |v_j|."""

import math

import pytest
import torch

from torch2iron_amd import model as gm
from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
D = 128
NAN = float("nan")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=g.device, generator=g).to(BF16)


def _attend(q, k, v, seen):
    """float64: q [R, D], k / v [K, D], seen bool [R, K] -> out, sum p |v|; an empty row is zero."""
    x = (q.double() @ k.double().T.contiguous()) / math.sqrt(D)
    x = x.masked_fill(~seen, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300)).masked_fill(~seen, 0.0)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return w @ v.double(), w @ v.double().abs()


def _check(out, ref, mag, what=""):
    err = (out.double() - ref).abs()
    tol = 2.0 ** -8 * (mag + 3 * ref.abs()) + 2e-4 * (mag.max() if mag.numel() else 0.0)
    assert torch.isfinite(out.double()).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: worst {(err - tol).max():.3e} over, error {err.max():.3e}"


# ---- packed prompts ----
# (hq, hkv, cap, lengths, starts, cache_rows or None, cache rows)
PACKED = [
    (16, 8, 64, [1], [0], None, 1),
    (2, 1, 300, [1, 1, 1], [0, 63, 299], None, 3),
    (16, 8, 320, [43, 7, 1], [0, 0, 0], None, 3),
    (8, 8, 400, [0, 129, 0, 64, 128], [0, 0, 5, 0, 127], None, 5),
    (8, 1, 200, [63, 64, 65], [1, 0, 64], None, 3),
    (7, 1, 777, [100, 0, 333], [3, 0, 444], None, 3),
    (24, 8, 257, [31, 257], [100, 0], None, 2),
    (40, 4, 150, [13, 77], [60, 0], None, 2),
    (32, 8, 1100, [300, 1, 2], [800, 1099, 500], [4, 0, 2], 6),
    (4, 1, 5000, [3], [4990], None, 1),                       # few rows over a long context: parts
    (16, 2, 9000, [40, 1, 1, 17], [8960, 8999, 5, 3000], [3, 1, 0, 2], 4),
    (16, 8, 2100, [2085], [15], None, 1),
]
PACKED_IDS = [f"{c[0]}-{c[1]}-" + "_".join(map(str, c[3])) for c in PACKED]


def _packed_case(gpu, hq, hkv, cap, lengths, starts, cache_rows, n_cache, seed=0):
    g = _gen(gpu, seed + cap + hq)
    plan = ops.PackedPlan(lengths, hq, hkv, cap, gpu, starts=starts, cache_rows=cache_rows, n_cache_rows=n_cache)
    q = _normal(g, plan.rows, hq, D)
    kc, vc = (_normal(g, n_cache, hkv, cap, D) for _ in range(2))
    for c in (kc, vc):                       # what no row attends holds NaN
        used = {r: s + n for n, s, r in zip(lengths, starts, plan.cache_rows) if n}
        for r in range(n_cache):
            c[r, :, used.get(r, 0):] = NAN
    return plan, q, kc, vc


def _packed_reference(plan, q, kc, vc):
    hq, hkv = plan.n_heads, plan.n_kv_heads
    ref = torch.zeros(plan.rows, hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(ref)
    for s, (n, start, row) in enumerate(zip(plan.lengths, plan.starts, plan.cache_rows)):
        if n == 0:
            continue
        a = plan.first_rows[s]
        seen = torch.arange(start + n, device=q.device) <= start + torch.arange(n, device=q.device)[:, None]
        for h in range(hq):
            kv = h // (hq // hkv)
            ref[a:a + n, h], mag[a:a + n, h] = _attend(q[a:a + n, h], kc[row, kv, :start + n], vc[row, kv, :start + n],
                                                       seen)
    return ref.view(plan.rows, -1), mag.view(plan.rows, -1)


@pytest.mark.parametrize("hq,hkv,cap,lengths,starts,cache_rows,n_cache", PACKED, ids=PACKED_IDS)
def test_packed_attention(gpu, hq, hkv, cap, lengths, starts, cache_rows, n_cache):
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, lengths, starts, cache_rows, n_cache)
    ref, mag = _packed_reference(plan, q, kc, vc)
    sums = torch.full((hq, plan.rows), 7.0, device=gpu)
    out = ops.packed_attention(q, plan, kc, vc, out_sums=sums)
    again = ops.packed_attention(q, plan, kc, vc, workspace=ops.Workspace())
    _check(out, ref, mag)
    assert torch.equal(out, again), "repeat calls differ"
    want = out.view(plan.rows, hq, D).double().sum(-1).T      # 128 fp32 additions of the rounded values
    bound = 128 * 2.0 ** -24 * out.view(plan.rows, hq, D).double().abs().sum(-1).T
    assert ((sums.double() - want).abs() <= bound + 1e-30).all()


def test_packed_attention_splits_and_merges(gpu):
    """The batches above whose plans split keys really do."""
    plans = [ops.PackedPlan(c[3], c[0], c[1], c[2], gpu, starts=c[4], cache_rows=c[5], n_cache_rows=c[6]) for c in PACKED]
    assert sum(p.n_parts > 0 for p in plans) >= 5 and sum(p.n_parts == 0 for p in plans) >= 5


def test_packed_equal_lengths_agree_with_the_batch_form(gpu):
    """Equal fresh prompts: the packed and the batch attention within their common tolerance of the truth."""
    b, t, hq, hkv, cap = 3, 150, 16, 8, 200
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, [t] * b, [0] * b, None, b)
    ref, mag = _packed_reference(plan, q, kc, vc)
    batch = ops.prefill_attention(q.view(b, t, hq, D).transpose(1, 2).contiguous(), 0, hkv, kc, vc)
    _check(ops.packed_attention(q, plan, kc, vc), ref, mag, "packed")
    _check(batch, ref, mag, "batch")


def test_packed_row_of_equal_values_is_exact(gpu):
    """Weights and normaliser are the same rounded numbers: constant values come back bit for bit."""
    plan, q, kc, vc = _packed_case(gpu, 8, 2, 700, [200, 5], [0, 650], None, 2)
    vc[:] = 1.375
    out = ops.packed_attention(q, plan, kc, vc)
    assert (out == 1.375).all()


def test_packed_large_scores(gpu):
    """Scores of tens, growing and falling along the keys: the running maximum follows."""
    hq, hkv, cap, n = 4, 2, 600, 555
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, [n], [0], None, 1)
    for ramp in (torch.linspace(0.0, 60.0, n, device=gpu), torch.linspace(60.0, 0.0, n, device=gpu)):
        k2 = kc.clone()
        k2[0, :, :n] = (ramp[:, None] * q[0, 0].float() / D).to(BF16)
        q2 = (q[:1, :1].float() * 12).expand(n, hq, D).to(BF16).contiguous()
        x = (q2[0, 0].double() @ k2[0, 0, :n].double().T.contiguous()) / math.sqrt(D)
        assert x.max() > 50
        ref, mag = _packed_reference(plan, q2, k2, vc)
        out = ops.packed_attention(q2, plan, k2, vc)
        # scores of up to ~70 in fp32: 128 products summed, 70 * 128 * 2^-24 = 5e-4 of a weight at most
        _check(out, ref, mag)


def test_packed_nan_stays_in_its_rows(gpu):
    """A NaN in one query row, also over split keys, reaches that row's heads alone."""
    for cap, lengths, starts in ((300, [150], [0]), (6000, [3], [5900])):
        plan, q, kc, vc = _packed_case(gpu, 4, 1, cap, lengths, starts, None, 1)
        clean = ops.packed_attention(q, plan, kc, vc)
        q[1, 2, 5] = NAN
        out = ops.packed_attention(q, plan, kc, vc).view(-1, 4, D)
        assert out[1, 2].isnan().all()
        out[1, 2] = clean.view(-1, 4, D)[1, 2]
        assert torch.equal(out.view_as(clean), clean)


@pytest.mark.parametrize("cap,lengths,starts", [(300, [150, 20], [0, 3]), (6000, [40], [5900]), (700, [3, 300], [600, 100])])
def test_what_a_mask_hides_stays_hidden(gpu, cap, lengths, starts):
    """Infinities and NaN in K and V of later rows of the same tile, also over split keys: rows that do
    not attend them are as without them, rows that do are what the definition gives."""
    hq, hkv = 8, 2
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, lengths, starts, None, len(lengths))
    clean, mag = _packed_reference(plan, q, kc, vc)
    sums = torch.zeros(hq, plan.rows, device=gpu)
    hit = torch.zeros(plan.rows, hq, dtype=torch.bool, device=gpu)
    for s, (n, start) in enumerate(zip(lengths, starts)):
        row = max(1, 2 * n // 3)
        kc[s, 0, start + row, 5] = NAN
        vc[s, 0, start + row - 1, 9] = float("inf")
        vc[s, 1, start + n - 1] = NAN
        a = plan.first_rows[s]
        hit[a + row - 1:a + n, :4] = True
        hit[a + n - 1, 4:] = True
    out = ops.packed_attention(q, plan, kc, vc, out_sums=sums).view(plan.rows, hq, D)
    ref, m = clean.view(plan.rows, hq, D), mag.view(plan.rows, hq, D)
    assert torch.isfinite(out[~hit].float()).all()
    _check(out[~hit], ref[~hit], m[~hit])
    for s, (n, start) in enumerate(zip(lengths, starts)):
        a, row = plan.first_rows[s], max(1, 2 * n // 3)
        assert (out[a + row - 1, :4, 9] == float("inf")).all() and out[a + row:a + n, :4].isnan().all()
        assert out[a + n - 1, 4:].isnan().all()
        rest = [d for d in range(D) if d != 9]
        _check(out[a + row - 1, :4][:, rest], ref[a + row - 1, :4][:, rest], m[a + row - 1, :4][:, rest])
    fine = ~hit
    want = out.double().sum(-1)
    bound = 128 * 2.0 ** -24 * out.double().abs().sum(-1)
    assert ((sums.T.double() - want).abs()[fine] <= bound[fine] + 1e-30).all()


@pytest.mark.parametrize("cap,ctx,n", [(200, [70, 3], 30), (4000, [3900], 64), (300, [200], 64)])
def test_a_sibling_s_infinity_stays_its_own(gpu, cap, ctx, n):
    """An infinity in one node's V and a NaN in another's K reach the nodes below them alone."""
    hq, hkv = (8, 2) if cap != 300 else (32, 4)
    q, parents, ctx_t, _, kc, vc, counts = _tree_case(gpu, hq, hkv, cap, ctx, n, None, "random")
    ref, mag = _tree_reference(q, parents, ctx, counts, kc, vc, cap)
    inf_node, nan_node = n // 2, n // 3
    for i, c in enumerate(ctx):
        vc[i, :, c + inf_node, 3] = float("inf")
        kc[i, :, c + nan_node, 7] = NAN
    out = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc).view(len(ctx), n, hq, D)
    for i in range(len(ctx)):
        for node, path in enumerate(_paths(parents[i].tolist())):
            o = out[i, node]
            if nan_node in path:
                assert o.isnan().all()
                continue
            if inf_node in path:
                assert (o[:, 3] == float("inf")).all()
                o = torch.cat((o[:, :3], o[:, 4:]), 1)
                _check(o, *(torch.cat((x[i, node][:, :3], x[i, node][:, 4:]), 1) for x in (ref, mag)))
                continue
            _check(o, ref[i, node], mag[i, node], f"sequence {i} node {node}")


@pytest.mark.parametrize("style", [ops.ROPE_HALVES, ops.ROPE_INTERLEAVED])
def test_packed_prep_has_the_bits_of_the_batch_form(gpu, style):
    hq, hkv, cap = 12, 4, 300
    lengths, starts, rows = [37, 0, 1, 120], [0, 9, 299, 77], [2, 4, 0, 3]
    g = _gen(gpu, 5)
    plan = ops.PackedPlan(lengths, hq, hkv, cap, gpu, starts=starts, cache_rows=rows, n_cache_rows=5)
    qkv = _normal(g, plan.rows, (hq + 2 * hkv) * D)
    qn, kn = ((0.9 + 0.2 * torch.rand(D, device=gpu, generator=g)).to(BF16) for _ in range(2))
    rope = gm.rope_table(D, cap, 1e6, gpu)
    kc, vc = (_normal(g, 5, hkv, cap, D) for _ in range(2))
    k2, v2 = kc.clone(), vc.clone()
    q = ops.packed_qk_rope_kv(qkv, plan, qn, kn, 1e-6, rope, kc, vc, rope_style=style)
    for s, (n, start, row) in enumerate(zip(lengths, starts, rows)):
        if n:
            a = plan.first_rows[s]
            q1 = ops.prefill_qk_rope_kv(qkv[a:a + n].contiguous(), 1, start, hq, hkv, qn, kn, 1e-6, rope, k2[row:row + 1],
                                        v2[row:row + 1], rope_style=style)
            assert torch.equal(q[a:a + n], q1[0].transpose(0, 1))
    assert torch.equal(kc, k2) and torch.equal(vc, v2)       # every other slot as it was


def test_packed_of_no_rows(gpu):
    plan = ops.PackedPlan([0, 0], 4, 2, 16, gpu)
    kc = torch.zeros(2, 2, 16, D, dtype=BF16, device=gpu)
    assert plan.rows == 0
    assert ops.packed_attention(torch.empty(0, 4, D, dtype=BF16, device=gpu), plan, kc, kc).shape == (0, 4 * D)


# ---- drafted trees ----

def _random_parents(b, n, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.tensor([[-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)] for _ in range(b)],
                     dtype=torch.int32)
    return p


def _paths(parents):
    """For each node the nodes above it and itself; a parent outside [0, node) makes a root."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


# (hq, hkv, cap, context lengths, nodes, counts or None, tree)
TREES = [
    (16, 8, 128, [0], 1, None, "random"),
    (2, 1, 200, [63, 64, 65], 8, None, "random"),
    (16, 8, 1088, [700], 8, None, "random"),
    (8, 8, 300, [0, 1, 200], 64, None, "random"),
    (8, 1, 700, [129, 600], 37, None, "chain"),
    (7, 1, 500, [400, 3], 26, None, "star"),
    (32, 8, 2000, [1936, 1000, 0], 64, None, "random"),
    (24, 8, 400, [100, 300, 7, 390], 13, [13, 0, 1, 5], "random"),
    (4, 2, 330, [-1, 300, 250, 330, 1], 31, [31, 31, 31, 0, 31], "random"),    # the first two outside the cache
    (16, 2, 9000, [8930, 10], 20, None, "odd"),
    (4, 1, 4000, [63, 3999], 1, None, "random"),
]
TREE_IDS = [f"{c[0]}-{c[1]}-cap{c[2]}-N{c[4]}-{c[6]}" for c in TREES]


def _tree_parents(kind, b, n, seed):
    if kind == "chain":
        return torch.arange(-1, n - 1, dtype=torch.int32).expand(b, n).contiguous()
    if kind == "star":
        return torch.tensor([[-1] + [0] * (n - 1)] * b, dtype=torch.int32)
    p = _random_parents(b, n, seed)
    if kind == "odd":                       # several roots, parents that no node may have
        p[:, 3], p[:, 7], p[:, 9], p[:, 11] = -5, 7, 12, 2**31 - 1
    return p


def _tree_case(gpu, hq, hkv, cap, ctx, n, counts, kind, seed=0):
    g = _gen(gpu, seed + cap + n)
    b = len(ctx)
    parents = _tree_parents(kind, b, n, seed + n)
    counts_l = [n] * b if counts is None else counts
    q = _normal(g, b, n, hq, D)
    kc, vc = (_normal(g, b, hkv, cap, D) for _ in range(2))
    for c in (kc, vc):
        for i in range(b):
            end = ctx[i] + counts_l[i] if ctx[i] >= 0 else 0
            c[i, :, end:] = NAN
    t = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    return q, parents.to(gpu), t(ctx), t(counts), kc, vc, counts_l


def _tree_reference(q, parents, ctx, counts, kc, vc, cap):
    b, n, hq, _ = q.shape
    hkv = kc.shape[1]
    ref = torch.zeros(b, n, hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(ref)
    for i in range(b):
        m, c = counts[i], ctx[i]
        if m == 0 or c < 0 or c + m > cap:
            continue
        seen = torch.zeros(m, c + m, dtype=torch.bool)
        seen[:, :c] = True
        for node, path in enumerate(_paths(parents[i].tolist()[:m])):
            seen[node, [c + j for j in path]] = True
        seen = seen.to(q.device)
        for h in range(hq):
            kv = h // (hq // hkv)
            ref[i, :m, h], mag[i, :m, h] = _attend(q[i, :m, h], kc[i, kv, :c + m], vc[i, kv, :c + m], seen)
    return ref, mag


@pytest.mark.parametrize("hq,hkv,cap,ctx,n,counts,kind", TREES, ids=TREE_IDS)
def test_tree_attention(gpu, hq, hkv, cap, ctx, n, counts, kind):
    q, parents, ctx_t, counts_t, kc, vc, counts_l = _tree_case(gpu, hq, hkv, cap, ctx, n, counts, kind)
    ref, mag = _tree_reference(q, parents, ctx, counts_l, kc, vc, cap)
    b = len(ctx)
    out = torch.full((b * n, hq * D), 7.0, dtype=BF16, device=gpu)
    got = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t, out=out).view(b, n, hq, D)
    again = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t, workspace=ops.Workspace())
    for i in range(b):
        _check(got[i, :counts_l[i]], ref[i, :counts_l[i]], mag[i, :counts_l[i]], f"sequence {i}")
        assert (got[i, counts_l[i]:] == 7.0).all(), "rows behind the last node were written"
        assert torch.equal(got[i, :counts_l[i]], again.view(b, n, hq, D)[i, :counts_l[i]])


def test_tree_attention_of_a_chain_is_the_packed_attention(gpu):
    """A chain of nodes is a prompt chunk: both within the tolerance of one truth."""
    hq, hkv, cap, n, ctx = 16, 8, 900, 24, [500, 0, 876]
    q, parents, ctx_t, _, kc, vc, counts = _tree_case(gpu, hq, hkv, cap, ctx, n, None, "chain")
    ref, mag = _tree_reference(q, parents, ctx, counts, kc, vc, cap)
    plan = ops.PackedPlan([n] * 3, hq, hkv, cap, gpu, starts=ctx)
    _check(ops.tree_attention(q, parents, ctx_t, hkv, kc, vc).view_as(ref), ref, mag, "tree")
    _check(ops.packed_attention(q.view(-1, hq, D), plan, kc, vc).view_as(ref), ref, mag, "packed")


@pytest.mark.parametrize("style", [ops.ROPE_HALVES, ops.ROPE_INTERLEAVED])
def test_tree_prep(gpu, style):
    """Every node's q, k and v as the standalone norm + RoPE at its position gives them, k and v in its
    slot; other slots, rows behind a count and sequences that do not fit as they were."""
    hq, hkv, cap, n = 6, 2, 120, 17
    ctx, counts = [40, 0, 110, -3, 103], [17, 9, 17, 17, 17]
    b = len(ctx)
    g = _gen(gpu, 3)
    parents = _tree_parents("odd", b, n, 4)
    qkv = _normal(g, b * n, (hq + 2 * hkv) * D)
    qn, kn = ((0.9 + 0.2 * torch.rand(D, device=gpu, generator=g)).to(BF16) for _ in range(2))
    rope = gm.rope_table(D, cap, 1e6, gpu)
    kc, vc = (_normal(g, b, hkv, cap, D) for _ in range(2))
    k_ref, v_ref = kc.clone(), vc.clone()
    q_ref = torch.full((b, n, hq, D), 7.0, dtype=BF16, device=gpu)
    rows = qkv.view(b, n, hq + 2 * hkv, D)
    for i in range(b):
        if ctx[i] < 0 or ctx[i] + counts[i] > cap:
            continue
        for node, path in enumerate(_paths(parents[i].tolist())[:counts[i]]):
            ang = rope[ctx[i] + len(path) - 1:ctx[i] + len(path)].contiguous()
            q_ref[i, node] = ops.rmsnorm_rope(rows[i, node, :hq].contiguous(), qn, ang, 1e-6, rope_style=style)
            k_ref[i, :, ctx[i] + node] = ops.rmsnorm_rope(rows[i, node, hq:hq + hkv].contiguous(), kn, ang, 1e-6,
                                                          rope_style=style)
            v_ref[i, :, ctx[i] + node] = rows[i, node, hq + hkv:]
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    q = ops.tree_qk_rope_kv(qkv, parents.to(gpu), t(ctx), hq, hkv, qn, kn, 1e-6, rope, kc, vc, rope_style=style,
                            node_counts=t(counts), q_out=torch.full_like(q_ref, 7.0))
    assert torch.equal(q, q_ref) and torch.equal(kc, k_ref) and torch.equal(vc, v_ref)


def _commit_reference(tokens, parents, picks, ctx, counts, kc, vc, cap):
    b, n = tokens.shape
    path, m, nxt, out = torch.full((b, n), -1), [], [], []
    k, v = kc.clone(), vc.clone()
    for i in range(b):
        c = max(0, min(counts[i], n))
        if c == 0 or ctx[i] < 0 or ctx[i] + c > cap:
            m.append(0), nxt.append(-1), out.append(ctx[i])
            continue
        walk = [0]
        while True:
            kids = [j for j in range(c) if j > walk[-1] and parents[i][j] == walk[-1] and tokens[i][j] == picks[i][walk[-1]]]
            if not kids:
                break
            walk.append(kids[0])
        path[i, :len(walk)] = torch.tensor(walk)
        m.append(len(walk)), nxt.append(int(picks[i][walk[-1]])), out.append(ctx[i] + len(walk))
        for to, node in enumerate(walk):
            k[:, i, :, ctx[i] + to] = kc[:, i, :, ctx[i] + node]
            v[:, i, :, ctx[i] + to] = vc[:, i, :, ctx[i] + node]
    return path, m, nxt, out, k, v


COMMITS = [(1, 1, 1, 4, [3], None, "random", 2), (3, 2, 8, 40, [5, 32], None, "random", 1),
           (2, 4, 26, 90, [0, 64, 50, 80], [26, 26, 3, 26], "random", 2), (28, 8, 64, 80, [16, 0, 3], [64, 99, -2], "chain", 1),
           (1, 2, 30, 60, [-1, 31, 30, 2], None, "odd", 2), (2, 3, 64, 64, [0, 0], None, "star", 2)]


@pytest.mark.parametrize("layers,hkv,n,cap,ctx,counts,kind,vocab", COMMITS)
def test_tree_commit(gpu, layers, hkv, n, cap, ctx, counts, kind, vocab):
    """vocab 1: every child is right (the longest walks); more: some are."""
    b = len(ctx)
    g = _gen(gpu, n + cap)
    parents = _tree_parents(kind, b, n, 9)
    tokens, picks = (torch.randint(0, vocab, (b, n), generator=torch.Generator().manual_seed(s), dtype=torch.int32) for s in (1, 2))
    kc, vc = (_normal(g, layers, b, hkv, cap, D) for _ in range(2))
    ref = _commit_reference(tokens, parents.tolist(), picks, ctx, [n] * b if counts is None else counts, kc, vc, cap)
    t = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    path, m, nxt, out = ops.tree_commit(tokens.to(gpu), parents.to(gpu), picks.to(gpu), t(ctx), kc, vc, node_counts=t(counts))
    assert path.cpu().tolist() == ref[0].tolist()
    assert (m.tolist(), nxt.tolist(), out.tolist()) == ref[1:4]
    assert torch.equal(kc, ref[4]) and torch.equal(vc, ref[5])


def test_tree_calls_replayed_from_a_graph(gpu):
    """One captured prep + attention + commit serves steps with other contexts, trees and counts."""
    hq, hkv, cap, n, b, layers = 8, 2, 1500, 11, 3, 1
    g = _gen(gpu, 1)
    qn = kn = torch.ones(D, dtype=BF16, device=gpu)
    rope = gm.rope_table(D, cap, 1e6, gpu)
    s = {"qkv": _normal(g, b * n, (hq + 2 * hkv) * D), "parents": _random_parents(b, n, 0).to(gpu),
         "ctx": torch.zeros(b, dtype=torch.int32, device=gpu), "counts": torch.full((b,), n, dtype=torch.int32, device=gpu),
         "tokens": torch.zeros(b, n, dtype=torch.int32, device=gpu), "picks": torch.zeros(b, n, dtype=torch.int32, device=gpu)}
    cache0 = [_normal(g, layers, b, hkv, cap, D) for _ in range(2)]
    cache = [c.clone() for c in cache0]
    ws = ops.Workspace()

    def step(caches):
        k, v = caches
        q = ops.tree_qk_rope_kv(s["qkv"], s["parents"], s["ctx"], hq, hkv, qn, kn, 1e-6, rope, k[0], v[0], node_counts=s["counts"])
        o = ops.tree_attention(q, s["parents"], s["ctx"], hkv, k[0], v[0], node_counts=s["counts"], workspace=ws)
        return o, *ops.tree_commit(s["tokens"], s["parents"], s["picks"], s["ctx"], k, v, node_counts=s["counts"])

    step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(cache)
    for i, ctx in enumerate(([0, 700, 1489], [1200, 3, 64], [5, 6, 7])):
        s["qkv"].copy_(_normal(g, b * n, (hq + 2 * hkv) * D))
        s["parents"].copy_(_random_parents(b, n, 20 + i))
        s["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        s["counts"].copy_(torch.tensor([n, n - i, 1 + i], dtype=torch.int32))
        s["tokens"].random_(0, 2, generator=g)
        s["picks"].random_(0, 2, generator=g)
        for c, c0 in zip(cache, cache0):
            c.copy_(c0)
        graph.replay()
        torch.cuda.synchronize()
        twin = [c.clone() for c in cache0]
        want = step(twin)
        counts = s["counts"].tolist()
        for j in range(b):
            assert torch.equal(res[0].view(b, n, -1)[j, :counts[j]], want[0].view(b, n, -1)[j, :counts[j]])
        assert all(torch.equal(x, y) for x, y in zip(res[1:], want[1:]))
        assert all(torch.equal(x, y) for x, y in zip(cache, twin))


def test_wrappers_refuse(gpu):
    """Shapes, types and plans that do not fit raise before anything is launched."""
    plan, q, kc, vc = _packed_case(gpu, 4, 2, 32, [3, 5], [0, 1], None, 2)
    tq, parents, ctx, _, tk, tv, _ = _tree_case(gpu, 4, 2, 32, [5, 6], 4, None, "random")
    qkv, one = torch.zeros(8, 8 * D, dtype=BF16, device=gpu), torch.ones(D, dtype=BF16, device=gpu)
    rope = gm.rope_table(D, 32, 1e6, gpu)
    i8 = torch.zeros(2, 4, dtype=torch.int32, device=gpu)
    x, t = torch.zeros(2, 9, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    for call in (
            lambda: ops.packed_attention(q[:7].contiguous(), plan, kc, vc), lambda: ops.packed_attention(q.float(), plan, kc, vc),
            lambda: ops.packed_attention(q[:, :2].contiguous(), plan, kc, vc),
            lambda: ops.packed_attention(q, plan, kc[:, :, :31].contiguous(), vc[:, :, :31].contiguous()),
            lambda: ops.packed_attention(q, plan, kc[:1], vc[:1]), lambda: ops.packed_attention(q, plan, kc, vc, out=q[:2]),
            lambda: ops.packed_attention(q, plan, kc, vc, out_sums=torch.zeros(3, device=gpu)),
            lambda: ops.packed_attention(q.transpose(1, 2), plan, kc, vc),
            lambda: ops.packed_qk_rope_kv(qkv[:7], plan, one, one, 1e-6, rope, kc, vc),
            lambda: ops.packed_qk_rope_kv(qkv, plan, one, one, 1e-6, rope[:31], kc, vc),
            lambda: ops.packed_qk_rope_kv(qkv, plan, one, one[:64], 1e-6, rope, kc, vc),
            lambda: ops.packed_qk_rope_kv(qkv, plan, one, one, 0.0, rope, kc, vc),
            lambda: ops.tree_attention(tq, parents.long(), ctx, 2, tk, tv), lambda: ops.tree_attention(tq, parents, ctx[:1], 2, tk, tv),
            lambda: ops.tree_attention(tq, parents[:, :3].contiguous(), ctx, 2, tk, tv), lambda: ops.tree_attention(tq, parents, ctx, 3, tk, tv),
            lambda: ops.tree_attention(tq, parents, ctx, 2, tk[:, :, :3].contiguous(), tv[:, :, :3].contiguous()),
            lambda: ops.tree_attention(tq, parents, ctx, 2, tk, tv, node_counts=ctx[:1]),
            lambda: ops.tree_attention(tq, parents.view(-1), ctx, 2, tk, tv),
            lambda: ops.tree_qk_rope_kv(qkv[:7], parents, ctx, 4, 2, one, one, 1e-6, rope, tk, tv),
            lambda: ops.tree_qk_rope_kv(qkv, parents, ctx, 4, 2, one, one, 1e-6, rope[:9], tk, tv),
            lambda: ops.tree_commit(i8, parents, i8[:1], ctx, tk, tv), lambda: ops.tree_commit(i8, parents, i8, ctx, tk, tv[:, :1]),
            lambda: ops.tree_commit(i8, parents, i8, ctx, tk[:1], tv[:1]), lambda: ops.tree_commit(i8.float(), parents, i8, ctx, tk, tv),
            lambda: ops.token_logprobs(x.double(), t), lambda: ops.token_logprobs(x, t[:1]), lambda: ops.token_logprobs(x, t.long()),
            lambda: ops.token_logprobs(x, t, top_k=10), lambda: ops.token_logprobs(x, t, top_k=-1),
            lambda: ops.token_logprobs(x[0], t), lambda: ops.token_logprobs(x.T, torch.zeros(9, dtype=torch.int32, device=gpu)),
            lambda: ops.token_logprobs(x[:1].expand(2, 9), t), lambda: ops.token_logprobs(torch.zeros(2, 99, device=gpu), t, top_k=33)):
        with pytest.raises(ValueError):
            call()


def test_calls_on_another_stream(gpu):
    """Packed and tree attention on two streams at once, without a workspace of the caller's."""
    plan, q, kc, vc = _packed_case(gpu, 4, 1, 6000, [3], [5900], None, 1)
    tq, parents, ctx, _, tk, tv, _ = _tree_case(gpu, 4, 1, 6000, [5000], 20, None, "random")
    want = ops.packed_attention(q, plan, kc, vc), ops.tree_attention(tq, parents, ctx, 1, tk, tv)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.packed_attention(q, plan, kc, vc), ops.tree_attention(tq, parents, ctx, 1, tk, tv)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
