"""Infinities and NaN in V: they reach the rows that attend them and no other, at a bounded cost."""

import pytest
import torch
from test_gpu_ragged import D, _check, _packed_case, _packed_reference, _paths, _tree_case, _tree_reference

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _expect(value, seen):
    """What attended values of one dim leave: value [K] with zeros for the finite ones, seen bool [R, K]."""
    plus, minus, nan = ((seen & m).any(-1) for m in (value == INF, value == -INF, value.isnan()))
    out = torch.zeros(seen.shape[0], dtype=torch.float64, device=seen.device)
    out[plus], out[minus] = INF, -INF
    out[nan | (plus & minus)] = NAN
    return out


def _strew(v, first, last, g):
    """A few infinities and NaN over slots first .. last - 1 of v [K, D], the ends among them."""
    for k in [first, last - 1] + torch.randint(first, last, (5,), generator=g).tolist():
        d = torch.randint(0, D, (2,), generator=g).tolist()
        v[k, d[0]] = (INF, -INF, NAN)[int(torch.randint(0, 3, (1,), generator=g))]
        v[k, d[1]] = INF


def _compare(out, clean, ref, mag, values, seen):
    """out [R, H, D] of one kv head with strewn values, clean: without them."""
    bad = ~torch.isfinite(values)
    want = torch.stack([_expect(torch.where(bad[:, d], values[:, d], 0.0), seen) for d in range(D)], -1)[:, None]
    hit = (want != 0).expand_as(ref)                          # NaN != 0
    assert torch.equal(out[hit].double().nan_to_num(7.0, 8.0, 9.0), want.expand_as(ref)[hit].nan_to_num(7.0, 8.0, 9.0))
    _check(out[~hit], ref[~hit], mag[~hit])
    rows = ~(seen & bad.any(-1)).any(-1)
    assert torch.equal(out[rows], clean[rows]), "rows that attend none changed"


@pytest.mark.parametrize("hq,hkv,cap,lengths,starts", [
    (2, 2, 400, [300, 129], [0, 77]), (16, 2, 300, [150, 20], [0, 3]), (6, 1, 700, [3, 300, 1, 1], [600, 100, 0, 650]),
    (4, 1, 6000, [40], [5900]), (4, 1, 6000, [1, 64], [5999, 0])])
def test_packed(gpu, hq, hkv, cap, lengths, starts):
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, lengths, starts, None, len(lengths))
    ref, mag = (x.view(plan.rows, hq, D) for x in _packed_reference(plan, q, kc, vc))
    clean = ops.packed_attention(q, plan, kc, vc).view(plan.rows, hq, D)
    g = torch.Generator().manual_seed(cap + hq)
    for s, (n, start) in enumerate(zip(lengths, starts)):
        for h in range(hkv):
            if (s + h) % 2 == 0:
                _strew(vc[s, h], start if s else 0, start + n, g)
    sums = torch.zeros(hq, plan.rows, device=gpu)
    out = ops.packed_attention(q, plan, kc, vc, out_sums=sums).view(plan.rows, hq, D)
    per = hq // hkv
    for s, (n, start) in enumerate(zip(lengths, starts)):
        a = plan.first_rows[s]
        seen = torch.arange(start + n, device=gpu) <= start + torch.arange(n, device=gpu)[:, None]
        for h in range(hkv):
            at = (slice(a, a + n), slice(h * per, (h + 1) * per))
            _compare(out[at], clean[at], ref[at], mag[at], vc[s, h, :start + n].double(), seen)
    want, fine = out.double().sum(-1).T, torch.isfinite(out).all(-1).T
    bound = 128 * 2.0 ** -24 * out.double().abs().sum(-1).T
    assert ((sums.double() - want).abs()[fine] <= bound[fine] + 1e-30).all() and not torch.isfinite(sums[~fine]).any()


@pytest.mark.parametrize("hq,hkv,cap,ctx,n,counts", [
    (8, 2, 200, [70, 3], 30, [30, 11]), (4, 1, 4000, [3900], 64, None), (32, 4, 300, [200, 0], 64, [64, 40])])
def test_tree(gpu, hq, hkv, cap, ctx, n, counts):
    q, parents, ctx_t, counts_t, kc, vc, counts_l = _tree_case(gpu, hq, hkv, cap, ctx, n, counts, "random")
    ref, mag = _tree_reference(q, parents, ctx, counts_l, kc, vc, cap)
    run = lambda: ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t).view(ref.shape)  # noqa: E731
    clean = run()
    g = torch.Generator().manual_seed(cap)
    for i, (c, m) in enumerate(zip(ctx, counts_l)):
        _strew(vc[i, 0], c, c + m, g)
    out, per = run(), hq // hkv
    for i, (c, m) in enumerate(zip(ctx, counts_l)):
        seen = torch.zeros(m, c + m, dtype=torch.bool)
        seen[:, :c] = True
        for node, path in enumerate(_paths(parents[i].tolist()[:m])):
            seen[node, [c + j for j in path]] = True
        for h in range(hkv):
            at = (i, slice(0, m), slice(h * per, (h + 1) * per))
            _compare(out[at], clean[at], ref[at], mag[at], vc[i, h, :c + m].double(), seen.to(gpu))


@pytest.mark.parametrize("n", [1, 40])
def test_huge_values(gpu, n):
    """Values of 2^121 under scores that rise by less than the reference's slack: the weighted sum of 26 of them
    fits fp32 by weights of at most 1, not by weights of up to 2^8."""
    hq, hkv, cap, start = 4, 2, 128, 90 - n
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, [n], [start], None, 1)
    q[:] = 1.0
    kc[0, :, :64] = 0.0
    kc[0, :, 64:90] = 0.459                                  # scores of 5.2, 7.5 in log2
    vc[0, :, :90] = torch.where(vc[0, :, :90] < 0, -2.0 ** 121, 2.0 ** 121).to(vc.dtype)
    vc[0, :, :90, :3] = 2.0 ** 121
    ref, mag = _packed_reference(plan, q, kc, vc)
    out = ops.packed_attention(q, plan, kc, vc)
    assert torch.isfinite(out).all() and (out.view(n, hq, D)[..., :3] == 2.0 ** 121).all()
    _check(out, ref, mag)


def _time(f, n=5):
    f()
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(n + 1)]
    ev[0].record()
    for e in ev[1:]:
        f()
        e.record()
    torch.cuda.synchronize()
    return sorted(a.elapsed_time(b) for a, b in zip(ev, ev[1:]))[n // 2]


@pytest.mark.parametrize("slot", [0, 1999], ids=["first", "last"])
def test_cost_of_a_nan(gpu, slot):
    """One NaN, in a slot that every row attends or in the last one's own: the pass is run again, and 64 x 64
    products of one block done key by key; forming the rows again from all of their keys took 50 to 70 times
    the clean pass."""
    plan, q, kc, vc = _packed_case(gpu, 16, 8, 2048, [500], [1500], None, 1)
    run = lambda: ops.packed_attention(q, plan, kc, vc)  # noqa: E731
    clean = _time(run)
    vc[:, :, slot, 3] = NAN
    assert _time(run) <= 10 * clean


def test_cost_of_a_cache_of_nan(gpu):
    """Trees over caches whose V is NaN throughout: blocks that every row sees whole stay matrix products, so that
    the second pass costs about the first and the last two blocks' key by key products."""
    q, parents, ctx, _, kc, vc, _ = _tree_case(gpu, 16, 8, 8192, [8000 - 61 * i for i in range(16)], 26, None, "random")
    run = lambda: ops.tree_attention(q, parents, ctx, 8, kc, vc)  # noqa: E731
    clean = _time(run)
    vc[:] = NAN
    assert _time(run) <= 5 * clean
    assert run().isnan().all()
