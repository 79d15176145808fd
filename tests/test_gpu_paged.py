"""Attention over a cache in pages on the MI355X against plain float64 attention, slot by slot through the page table.

Tolerance of the attention, elementwise: weights w_j enter P . V rounded to bf16 (8 significant bits: neighbours in
[1, 2) are 2^-7 apart, so a rounding is off by at most 2^-8 relative) and are normalised by the sum of the rounded ones,
so an output moves by at most 2^-8 (sum p_j |v_j| + |out|); where a sequence's rows times Hq / Hkv are at most 128
weights have 16 bits, which the terms below cover.  The output's own rounding adds 2^-8 |out|.  fp32 scores of up to 40
over 128 terms and their sums, and second-order terms: 2e-4 of the largest sum p_j |v_j|, as for the packed rows over a
contiguous cache."""

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


class Case:
    """Sequences of ``lens`` rows behind ``ctx`` slots, their pages in no order in a pool that holds NaN elsewhere."""

    def __init__(self, dev, hq, hkv, page, lens, ctx, seed=0, spare=2, behind=0):
        g = _gen(dev, seed + 31 * hq + page)
        self.hq, self.hkv, self.page, self.lens, self.ctx = hq, hkv, page, lens, ctx
        need = [-(-(a + b) // page) for a, b in zip(lens, ctx)]
        order = torch.randperm(sum(need) + spare, device=dev, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32, device=dev)
        self.k, self.v = (torch.full((order.numel(), hkv, page, D), NAN, dtype=BF16, device=dev) for _ in range(2))
        self.slots = []                                   # (k, v) [Hkv, slots, D] of each sequence
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
            some = lens[i] + ctx[i] if lens[i] else 0
            kv = [_normal(g, hkv, some, D) for _ in range(2)]
            j = torch.arange(some, device=dev)
            where = self.table[i].long()[j // page], j % page
            for pool, x in zip((self.k, self.v), kv):
                pool[where[0], :, where[1]] = x.transpose(0, 1)
            self.slots.append(kv)
        self.rows = sum(lens) + behind
        self.row_starts = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
        self.ctx_dev = torch.tensor(ctx, dtype=torch.int32, device=dev)
        self.q = _normal(g, self.rows, hq, D)
        self.plan = ops.PagedPlan(self.rows, self.row_starts, self.ctx_dev, self.table, hq, hkv, page)

    def reference(self):
        ref = torch.zeros(self.rows, self.hq, D, dtype=torch.float64, device=self.q.device)
        mag = torch.zeros_like(ref)
        at = 0
        for n, start, (k, v) in zip(self.lens, self.ctx, self.slots):
            ahead = torch.ones(n, start + n, dtype=torch.bool, device=ref.device).triu(start + 1)
            for h in range(self.hq if n else 0):
                kh, vh = (x[h // (self.hq // self.hkv)].double() for x in (k, v))
                x = (self.q[at:at + n, h].double() @ kh.T.contiguous()) / math.sqrt(D)
                w = torch.softmax(x.masked_fill(ahead, -math.inf), -1)
                vz = vh.nan_to_num(0.0, 0.0, 0.0)
                ref[at:at + n, h], mag[at:at + n, h] = w @ vz, w @ vz.abs()
            at += n
        return ref.view(self.rows, -1), mag.view(self.rows, -1)


def _check(out, ref, mag, what=""):
    err = (out.double() - ref).abs()
    tol = 2.0 ** -8 * (mag + 2 * ref.abs()) + 2e-4 * (mag.max() if mag.numel() else 0.0)
    assert torch.isfinite(out.double()).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: worst {(err - tol).max():.3e} over, error {err.max():.3e}"


# (hq, hkv, page, lens, ctx)
CASES = [
    (16, 8, 16, [1], [0]),
    (2, 1, 16, [1, 1, 1], [0, 63, 64]),
    (16, 8, 32, [43, 7, 1], [0, 0, 0]),
    (8, 8, 64, [0, 129, 0, 64, 128], [0, 0, 5, 0, 127]),
    (8, 1, 256, [63, 64, 65], [1, 0, 64]),
    (7, 1, 16, [100, 0, 333], [3, 0, 444]),
    (24, 8, 128, [31, 257], [100, 0]),
    (40, 4, 16, [13, 77], [60, 0]),
    (32, 8, 16, [300, 1, 2], [800, 1099, 500]),
    (4, 1, 16, [3], [4990]),                                   # few rows over a long context: parts
    (16, 2, 32, [40, 1, 1, 17], [8960, 8999, 5, 3000]),
    (16, 8, 1024, [2085], [15]),
    (16, 8, 16, [5] * 16, [901 + 200 * i for i in range(16)]),
    (32, 8, 64, [1] * 70, [37 * i for i in range(70)]),
    (150, 1, 16, [2, 1], [30, 200]),                           # more q heads a kv head than a tile has pairs
    (32, 8, 64, [1, 40, 2] + [1] * 70, [9000, 4000, 100] + [11 * i for i in range(70)]),   # many tiles, the longest cut
]
IDS = [f"{c[0]}-{c[1]}-p{c[2]}-" + "_".join(map(str, c[3][:6])) for c in CASES]


@pytest.mark.parametrize("hq,hkv,page,lens,ctx", CASES, ids=IDS)
def test_paged_attention(gpu, hq, hkv, page, lens, ctx):
    c = Case(gpu, hq, hkv, page, lens, ctx)
    ref, mag = c.reference()
    sums = torch.full((hq, c.rows), 7.0, device=gpu)
    out = ops.paged_attention(c.q, c.plan, c.k, c.v, out_sums=sums)
    again = ops.paged_attention(c.q, c.plan, c.k, c.v, workspace=ops.Workspace())
    _check(out, ref, mag)
    assert torch.equal(out, again), "repeat calls differ"
    want = out.view(c.rows, hq, D).double().sum(-1).T          # 128 fp32 additions of the rounded values
    bound = 128 * 2.0 ** -24 * out.view(c.rows, hq, D).double().abs().sum(-1).T
    assert ((sums.double() - want).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("longest", [90, 9000], ids=["whole", "cut"])
def test_more_tiles_than_the_plan_has_threads(gpu, longest):
    n = 2500
    c = Case(gpu, 2, 1, 16, [1 + i % 2 for i in range(n)], [longest if i == 1234 else i % 40 for i in range(n)])
    out = ops.paged_attention(c.q, c.plan, c.k, c.v)
    _check(out, *c.reference())


def test_more_kv_heads_than_workgroups_run_at_once(gpu):
    c = Case(gpu, 520, 520, 16, [3, 1, 2], [40, 700, 7])
    _check(ops.paged_attention(c.q, c.plan, c.k, c.v), *c.reference())


def test_as_many_sequences_as_a_plan_takes(gpu):
    n = 4096
    c = Case(gpu, 1, 1, 16, [i % 3 for i in range(n)], [i % 70 for i in range(n)])
    _check(ops.paged_attention(c.q, c.plan, c.k, c.v), *c.reference())


def test_values_behind_a_mask_stay_there(gpu):
    """NaN and infinities in slots that a row does not attend do not reach it; rows that attend them take them."""
    for bad in (NAN, math.inf, -math.inf):
        for lens, ctx, hq, hkv in (([200, 9], [70, 3], 16, 8), ([1], [3000], 4, 1)):
            c = Case(gpu, hq, hkv, 16, lens, ctx)
            clean = ops.paged_attention(c.q, c.plan, c.k, c.v)
            last = lens[0] + ctx[0] - 1                    # the last slot: its own row alone attends it
            c.v[int(c.table[0, last // 16]), :, last % 16, 5] = bad
            out = ops.paged_attention(c.q, c.plan, c.k, c.v)
            row = lens[0] - 1
            other = torch.arange(c.rows, device=gpu) != row
            assert torch.equal(out[other], clean[other])
            mine, was = out[row].view(hq, D), clean[row].view(hq, D)
            assert not torch.isfinite(mine[:, 5].float()).any()
            assert torch.equal(torch.isfinite(mine.float()).sum(-1), torch.full((hq,), D - 1, device=gpu))
            keep = torch.arange(D, device=gpu) != 5
            assert (mine[:, keep].float() - was[:, keep].float()).abs().max() < 0.05


def test_single_tokens_and_drafts_among_long_chunks(gpu):
    """The form of narrow tiles among wide ones: values, values behind a mask, pages outside the pool."""
    lens, ctx, hq, hkv = [300, 1, 5, 1, 3, 7], [800, 1099, 500, 0, 31, 2050], 32, 8
    for page in (16, 128):
        c = Case(gpu, hq, hkv, page, lens, ctx)
        clean = ops.paged_attention(c.q, c.plan, c.k, c.v)
        ref, mag = c.reference()
        _check(clean, ref, mag)
        start = torch.tensor([0] + lens).cumsum(0).tolist()
        for s in (2, 5):                                   # drafts: the last row alone attends the last slot
            last = lens[s] + ctx[s] - 1
            was = c.v[int(c.table[s, last // page]), :, last % page, 5].clone()
            for bad in (NAN, math.inf):
                c.v[int(c.table[s, last // page]), :, last % page, 5] = bad
                out = ops.paged_attention(c.q, c.plan, c.k, c.v)
                row = start[s + 1] - 1
                at = torch.arange(c.rows, device=gpu)
                own = (at >= start[s]) & (at <= row)
                assert torch.equal(out[~own], clean[~own])
                # Rows that share a tile with such a value are formed again, with fp32 weights on that block (and
                # two bf16 words relative to another maximum on the others), where the clean call took two words
                # throughout: each is within the tolerance of the reference (errors of 2^-17 before the output's
                # rounding), but not the other's bits.
                _check(out[own & (at != row)], ref[own & (at != row)], mag[own & (at != row)])
                mine = torch.isfinite(out[row].view(hq, D).float())
                assert not mine[:, 5].any() and torch.equal(mine.sum(-1), torch.full((hq,), D - 1, device=gpu))
            c.v[int(c.table[s, last // page]), :, last % page, 5] = was
        for s in (1, 4):
            was = int(c.table[s, 0])
            c.table[s, 0] = c.k.shape[0]
            out = ops.paged_attention(c.q, c.plan, c.k, c.v)
            mine = (torch.arange(c.rows, device=gpu) >= start[s]) & (torch.arange(c.rows, device=gpu) < start[s + 1])
            assert torch.isnan(out[mine]).all() and torch.equal(out[~mine], clean[~mine])
            c.table[s, 0] = was


def test_sequences_without_slots_and_rows_of_nobody(gpu):
    """A context below zero, or rows past the pages: zero rows, nothing written; rows behind the last sequence and
    row_starts that do not ascend: nothing at all."""
    c = Case(gpu, 8, 4, 16, [3, 40, 2, 5], [20, 100, 7, 30], behind=3)
    ref, mag = c.reference()
    cap = c.table.shape[1] * 16
    qkv = _normal(_gen(gpu, 1), c.rows, (8 + 2 * 4) * D)
    norm, rope = torch.ones(D, dtype=BF16, device=gpu), gm.rope_table(D, cap, 1e6, gpu)
    for ctx in (-1, -2**31, cap - 39, cap, 2**31 - 1):
        c.ctx_dev[1] = ctx
        c.plan.refresh()
        out = torch.full((c.rows, 8 * D), 3.0, dtype=BF16, device=gpu)
        ops.paged_attention(c.q, c.plan, c.k, c.v, out=out)
        _check(out[:3], ref[:3], mag[:3])
        _check(out[43:50], ref[43:50], mag[43:50])
        assert (out[3:43] == 0).all() and (out[50:] == 3.0).all()
        k, v = c.k.clone(), c.v.clone()
        q = torch.full((c.rows, 8, D), 3.0, dtype=BF16, device=gpu)
        ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, rope, k, v, q_out=q)
        assert (q[3:43] == 3.0).all() and (q[50:] == 3.0).all() and (q[:3] != 3.0).any()
        used = c.table[1, :9].long()
        assert torch.equal(k[used].nan_to_num(9.0), c.k[used].nan_to_num(9.0))
        assert torch.equal(v[used].nan_to_num(9.0), c.v[used].nan_to_num(9.0))
    c.ctx_dev[1] = 100
    for starts in ([0, 3, 2, 45, 50], [-1, 3, 43, 45, 50], [0, 3, 43, 45, 54]):
        c.row_starts.copy_(torch.tensor(starts, dtype=torch.int32))
        c.plan.refresh()
        out = torch.full((c.rows, 8 * D), 3.0, dtype=BF16, device=gpu)
        assert (ops.paged_attention(c.q, c.plan, c.k, c.v, out=out) == 3.0).all()


@pytest.mark.parametrize("starts", [[0, 3, 2, 45, 50], [-1, 3, 43, 45, 50], [0, 3, 43, 45, 54], [0, 50, 3, 45, 50]])
def test_row_starts_that_do_not_ascend_write_nothing(gpu, starts):
    c = Case(gpu, 8, 4, 16, [3, 40, 2, 5], [20, 100, 7, 30], behind=3)
    c.row_starts.copy_(torch.tensor(starts, dtype=torch.int32))
    c.plan.refresh()
    qkv = _normal(_gen(gpu, 1), c.rows, (8 + 2 * 4) * D)
    norm, rope = torch.ones(D, dtype=BF16, device=gpu), gm.rope_table(D, c.table.shape[1] * 16, 1e6, gpu)
    k, v = c.k.clone(), c.v.clone()
    q = torch.full((c.rows, 8, D), 3.0, dtype=BF16, device=gpu)
    ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, rope, k, v, q_out=q)
    assert (q == 3.0).all()
    assert torch.equal(k.nan_to_num(9.0), c.k.nan_to_num(9.0)) and torch.equal(v.nan_to_num(9.0), c.v.nan_to_num(9.0))


def test_rows_that_start_behind_the_first(gpu):
    """Rows before the first sequence's are no sequence's."""
    c = Case(gpu, 8, 4, 16, [3, 5], [20, 33], behind=4)
    ref, mag = c.reference()
    c.row_starts += 4
    c.plan.refresh()
    out = torch.full((c.rows, 8 * D), 3.0, dtype=BF16, device=gpu)
    q = c.q.roll(4, 0)
    ops.paged_attention(q, c.plan, c.k, c.v, out=out)
    _check(out[4:], ref[:8], mag[:8])
    assert (out[:4] == 3.0).all()


@pytest.mark.parametrize("lens,ctx", [([200, 9], [70, 3]), ([1, 2], [3000, 40])], ids=["whole", "parts"])
def test_pages_outside_the_pool(gpu, lens, ctx):
    """Their sequence's rows that attend them are NaN, the other sequences' as they were; a row to be written
    there writes its q alone."""
    c = Case(gpu, 16, 8, 16, lens, ctx)
    clean = ops.paged_attention(c.q, c.plan, c.k, c.v)
    last = lens[0] + ctx[0] - 1
    qkv = _normal(_gen(gpu, 1), c.rows, (16 + 2 * 8) * D)
    norm, rope = torch.ones(D, dtype=BF16, device=gpu), gm.rope_table(D, c.table.shape[1] * 16, 1e6, gpu)
    k0, v0 = c.k.clone(), c.v.clone()
    q0 = ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, rope, k0, v0)
    for bad in (-1, c.k.shape[0], 2**31 - 1, -2**31):
        was = int(c.table[0, last // 16])
        c.table[0, last // 16] = bad
        sums = torch.zeros(16, c.rows, device=gpu)
        out = ops.paged_attention(c.q, c.plan, c.k, c.v, out_sums=sums)
        assert torch.isnan(out[lens[0] - 1]).all() and torch.isnan(sums[:, lens[0] - 1]).all()
        assert torch.equal(out[lens[0]:], clean[lens[0]:])
        k, v = c.k.clone(), c.v.clone()
        q = ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, rope, k, v)
        assert torch.equal(q, q0)
        keep = torch.arange(c.k.shape[0], device=gpu) != was
        assert torch.equal(k[keep].nan_to_num(9.0), k0[keep].nan_to_num(9.0))
        assert torch.equal(k[was].nan_to_num(9.0), c.k[was].nan_to_num(9.0))
        c.table[0, last // 16] = was
    assert torch.equal(ops.paged_attention(c.q, c.plan, c.k, c.v), clean)


@pytest.mark.parametrize("style", [ops.ROPE_HALVES, ops.ROPE_INTERLEAVED])
def test_write_has_the_packed_bits(gpu, style):
    """q, and k and v in their slots, as the packed rows' write into a contiguous cache."""
    lens, ctx, hq, hkv, page = [1, 40, 0, 5, 1], [17, 3, 9, 63, 0], 10, 2, 32
    c = Case(gpu, hq, hkv, page, lens, ctx)
    cap = c.table.shape[1] * page
    g = _gen(gpu, 5)
    qkv = _normal(g, c.rows, (hq + 2 * hkv) * D)
    qn, kn = _normal(g, D), _normal(g, D)
    rope = gm.rope_table(D, cap, 1e6, gpu)
    plan = ops.PackedPlan(lens, hq, hkv, cap, gpu, starts=ctx)
    kc, vc = (torch.zeros(len(lens), hkv, cap, D, dtype=BF16, device=gpu) for _ in range(2))
    want = ops.packed_qk_rope_kv(qkv, plan, qn, kn, 1e-6, rope, kc, vc, rope_style=style)
    k0, v0 = c.k.clone(), c.v.clone()
    got = ops.paged_qk_rope_kv(qkv, c.plan, qn, kn, 1e-6, rope, c.k, c.v, rope_style=style)
    assert torch.equal(got, want)
    for s, (n, start) in enumerate(zip(lens, ctx)):
        j = torch.arange(start, start + n, device=gpu)
        at = c.table[s].long()[j // page], j % page
        for pool, was, cache in ((c.k, k0, kc), (c.v, v0, vc)):
            assert torch.equal(pool[at[0], :, at[1]], cache[s, :, j].transpose(0, 1))
            was[at[0], :, at[1]] = pool[at[0], :, at[1]]
    for pool, was in ((c.k, k0), (c.v, v0)):               # no other place is touched
        assert torch.equal(pool.nan_to_num(9.0), was.nan_to_num(9.0))


def test_shared_pages(gpu):
    """Two sequences over the same first pages."""
    c = Case(gpu, 8, 2, 16, [4, 4], [64, 64])
    c.table[1, :4] = c.table[0, :4]
    for i in range(2):
        c.slots[1][i][:, :64] = c.slots[0][i][:, :64]
    _check(ops.paged_attention(c.q, c.plan, c.k, c.v), *c.reference())


def test_pools_past_32_bit_offsets(gpu):
    """A pool of over 4 GB in bytes: its last pages are the ones in use."""
    page, hkv = 64, 8
    n = (1 << 32) // (page * hkv * D * 2) + 3
    c = Case(gpu, 16, hkv, page, [3, 1], [200, 500])
    ref, mag = c.reference()
    small = c.k.shape[0]
    pools = []
    for x in (c.k, c.v):
        big = torch.empty(n, hkv, page, D, dtype=BF16, device=gpu)
        big[:small].fill_(NAN)
        big[n - small:] = x
        pools.append(big)
    c.table[c.table >= 0] += n - small
    _check(ops.paged_attention(c.q, c.plan, *pools), ref, mag)
    qkv = _normal(_gen(gpu, 1), c.rows, (16 + 2 * hkv) * D)
    norm, rope = torch.ones(D, dtype=BF16, device=gpu), gm.rope_table(D, c.table.shape[1] * page, 1e6, gpu)
    ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, rope, *pools)
    last = int(c.table[1, 500 // page])
    assert torch.equal(pools[1][last, :, 500 % page].reshape(-1), qkv[3, (16 + hkv) * D:])
    assert torch.isnan(pools[0][:small]).all()


def test_captured_step_serves_later_ones(gpu):
    """Plan, write and attention in one graph, replayed over growing contexts, new pages and other splits of the rows,
    with eager work between, against the eager calls on the same state."""
    hq, hkv, page = 16, 8, 16
    lens, ctx = [1, 5, 1, 0], [15, 1000, 300, 0]
    c = Case(gpu, hq, hkv, page, lens, [x + 64 for x in ctx])
    c.ctx_dev.copy_(torch.tensor(ctx, dtype=torch.int32))
    c.k.nan_to_num_(0.5)
    c.v.nan_to_num_(0.25)
    cap = c.table.shape[1] * page
    g = _gen(gpu, 9)
    qkv = _normal(g, c.rows, (hq + 2 * hkv) * D)
    norm, rope = _normal(g, D), gm.rope_table(D, cap, 1e6, gpu)
    k2, v2 = c.k.clone(), c.v.clone()
    ws, out = ops.Workspace(), torch.zeros(c.rows, hq * D, dtype=BF16, device=gpu)
    q = torch.zeros(c.rows, hq, D, dtype=BF16, device=gpu)

    def step(k, v, plan, q, out, ws=None):
        plan.refresh()
        ops.paged_qk_rope_kv(qkv, plan, norm, norm, 1e-6, rope, k, v, q_out=q)
        ops.paged_attention(q, plan, k, v, out=out, workspace=ws)

    eager_plan = ops.PagedPlan(c.rows, c.row_starts, c.ctx_dev, c.table, hq, hkv, page)
    k1, v1 = c.k.clone(), c.v.clone()
    step(c.k, c.v, c.plan, q, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c.k, c.v, c.plan, q, out, ws)
    c.k.copy_(k1)
    c.v.copy_(v1)
    want_q, want = torch.zeros_like(q), torch.zeros_like(out)
    for i, starts in enumerate(([0, 1, 6, 7, 7], [0, 1, 6, 7, 7], [0, 0, 3, 7, 7], [0, 7, 7, 7, 7], [0, 1, 3, 6, 7])):
        c.row_starts.copy_(torch.tensor(starts, dtype=torch.int32))
        graph.replay()
        step(k2, v2, eager_plan, want_q, want)
        torch.cuda.synchronize()
        # bits: in the last replay sequence 2 has outgrown its pages, and its rows are NaN on both sides
        assert torch.equal(q, want_q) and torch.equal(out.view(torch.int16), want.view(torch.int16)), f"replay {i}"
        assert torch.isfinite(out[:6 if i < 4 else 3].float()).all()
        assert torch.equal(c.k, k2) and torch.equal(c.v, v2)
        c.ctx_dev[:3] += torch.tensor([1, 3, 17], dtype=torch.int32, device=gpu)
        qkv.copy_(_normal(g, *qkv.shape))


def test_calls_on_another_stream(gpu):
    c = Case(gpu, 16, 8, 16, [2, 30], [1000, 40])
    ref, mag = c.reference()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        plan = ops.PagedPlan(c.rows, c.row_starts, c.ctx_dev, c.table, 16, 8, 16)
        a = ops.paged_attention(c.q, plan, c.k, c.v)
        b = ops.paged_attention(c.q, c.plan, c.k, c.v)
    other.synchronize()
    _check(a, ref, mag)
    assert torch.equal(a, b)


def test_calls_side_by_side(gpu):
    """Two streams at once, each with its own workspace."""
    cases = [Case(gpu, 16, 8, 16, [1] * 8, [1500 + 100 * i for i in range(8)], seed=s) for s in range(2)]
    want = [ops.paged_attention(c.q, c.plan, c.k, c.v) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    ws = [ops.Workspace() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s, w in zip(cases, streams, ws):
            with torch.cuda.stream(s):
                got.append(ops.paged_attention(c.q, c.plan, c.k, c.v, workspace=w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(gpu):
    c = Case(gpu, 8, 4, 16, [0, 0], [5, 0])
    assert ops.paged_attention(c.q, c.plan, c.k, c.v).shape == (0, 8 * D)
    c.plan.refresh()


def test_wrapper_refusals(gpu):
    c = Case(gpu, 8, 4, 16, [2, 3], [5, 20])
    args = lambda **kw: {**dict(rows=c.rows, row_starts=c.row_starts, context_lens=c.ctx_dev, page_table=c.table,  # noqa: E731
                                n_heads=8, n_kv_heads=4, page_slots=16), **kw}
    for kw, what in ((dict(row_starts=c.row_starts[:-1].contiguous()), "row_starts must hold"),
                     (dict(context_lens=c.ctx_dev.long()), "int32"), (dict(context_lens=c.ctx_dev.cpu()), "GPU tensor"),
                     (dict(page_table=c.table[0]), "page_table"), (dict(page_table=c.table[:, ::2]), "contiguous"),
                     (dict(n_heads=9), "unsupported"), (dict(n_heads=2048, n_kv_heads=1), "unsupported"),
                     (dict(page_slots=48), "power of two"), (dict(page_slots=8), "power of two"),
                     (dict(page_slots=131072), "power of two"), (dict(rows=-1), "unsupported"), (dict(rows=2.5), "integers"),
                     (dict(rows=2**24), "too large")):
        with pytest.raises(ValueError, match=what):
            ops.PagedPlan(**args(**kw))
    many = torch.zeros(4097, 1, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="too large"):
        ops.PagedPlan(5, torch.zeros(4098, dtype=torch.int32, device=gpu), many[:, 0].contiguous(), many, 8, 4, 16)
    long = torch.zeros(1, 2**19 + 1, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="8388608"):
        ops.PagedPlan(5, torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu), long, 8, 4, 16)
    for q, k, v in ((c.q[:-1], c.k, c.v), (c.q.float(), c.k, c.v), (c.q, c.k[:, :2].contiguous(), c.v), (c.q, c.k, c.v[:-1]),
                    (c.q, c.k.transpose(1, 2), c.v), (c.q, c.k.float(), c.v), (c.q[..., :64].contiguous(), c.k, c.v)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, c.plan, k, v)
    with pytest.raises(ValueError, match="out must be"):
        ops.paged_attention(c.q, c.plan, c.k, c.v, out=torch.empty(c.rows, 7 * D, dtype=BF16, device=gpu))
    qkv, norm = torch.zeros(c.rows, 16 * D, dtype=BF16, device=gpu), torch.ones(D, dtype=BF16, device=gpu)
    with pytest.raises(ValueError, match="rope table"):
        ops.paged_qk_rope_kv(qkv, c.plan, norm, norm, 1e-6, gm.rope_table(D, 16, 1e6, gpu), c.k, c.v)
    with pytest.raises(ValueError, match="qkv must be"):
        ops.paged_qk_rope_kv(qkv[:-1], c.plan, norm, norm, 1e-6, gm.rope_table(D, 1024, 1e6, gpu), c.k, c.v)


@pytest.mark.parametrize("rows", [33, 40, 200])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2)])
def test_more_rows_than_a_sequence_has_slots(gpu, hq, hkv, rows):
    """Rows past everything that the table has: zero rows and sums, whatever the context; the others do not notice."""
    c = Case(gpu, hq, hkv, 16, [3, rows, 1], [20, 0, 7])
    ref, mag = c.reference()
    table = c.table[:, :2].contiguous()                    # 32 slots a sequence
    for ctx in (0, 5, -1):
        c.ctx_dev[1] = ctx
        plan = ops.PagedPlan(c.rows, c.row_starts, c.ctx_dev, table, hq, hkv, 16)
        out = torch.full((c.rows, hq * D), 3.0, dtype=BF16, device=gpu)
        sums = torch.full((hq, c.rows), 3.0, device=gpu)
        ops.paged_attention(c.q, plan, c.k, c.v, out=out, out_sums=sums)
        assert (out[3:-1] == 0).all() and (sums[:, 3:-1] == 0).all()
        _check(out[:3], ref[:3], mag[:3])
        _check(out[-1:], ref[-1:], mag[-1:])
