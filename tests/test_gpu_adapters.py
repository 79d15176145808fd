"""Adapters of many requests beside a projection on the MI355X against the definition in float64, row by row.

Tolerance, elementwise, of y + d with d = sum_r b_r h_r, h = scale sum_k a_k x_k: products of bf16 are exact in fp32, so
h is off by at most K 2^-24 sum |a x| |scale| and by its two bf16 words' rounding, each 2^-8 of what it rounds: 2^-16 |h|; the second
sum adds 2R 2^-24 sum |b h|; the result's rounding 2^-8 of itself.  SwiGLU: silu's slope is at most 1.1, so errors eg, eu
of gate and up make 1.1 eg |up| + |silu(gate)| eu + 1.1 eg eu, and fp32 exponential, division and product 2^-20 of the value."""

import pytest
import torch

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
NAN = float("nan")


def _make(gpu, k, widths, paired, rank, pool, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + k + rank)
    n, parts = sum(widths), 2 if paired else len(widths)
    a = (torch.randn(pool, parts, rank, k, device=gpu, generator=g) / k ** 0.5).to(BF16)
    b = (torch.randn(pool, n, rank, device=gpu, generator=g) / rank ** 0.5).to(BF16)
    scales = 0.25 + torch.rand(pool, device=gpu, generator=g)
    return g, a, b, scales, ops.Adapters(a, b, scales, widths=None if paired else widths, paired=paired)


def _reference(y, x, a, b, scales, widths, paired, ids):
    """float64 y + d, and the bound of the error of it before it is rounded."""
    out, err = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    k, rank = x.shape[1], a.shape[2]
    for i in set(ids.tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        rows = (ids == i).nonzero()[:, 0]
        xs, s, col = x[rows].double(), float(scales[i]), 0
        for part in range(a.shape[1]):
            aa = a[i, part].double()
            h, mag = s * (xs @ aa.T), abs(s) * (xs.abs() @ aa.abs().T)
            eh = k * 2.0 ** -24 * mag + 2.0 ** -16 * h.abs()
            cols = torch.arange(part, y.shape[1], 2) if paired else torch.arange(col, col + widths[part])
            cols = cols.to(y.device)
            col += 0 if paired else widths[part]
            bb = b[i, cols].double()
            at = rows[:, None], cols
            out[at] += h @ bb.T
            err[at] += eh @ bb.abs().T + 2 * rank * 2.0 ** -24 * ((h.abs() + eh) @ bb.abs().T) + 2.0 ** -24 * out[at].abs()
    return out, err


def _check(out, ref, err):
    d = (out.double() - ref).abs()
    tol = err + 2.0 ** -8 * (ref.abs() + err)
    assert (d <= tol).all(), f"{(d - tol).max():.3e} over, error {d.max():.3e}"


def _swiglu(ref, err):
    g, u, eg, eu = ref[:, 0::2], ref[:, 1::2], err[:, 0::2], err[:, 1::2]
    s = torch.nn.functional.silu(g)
    r = s * u
    return r, 1.1 * eg * u.abs() + s.abs() * eu + 1.1 * eg * eu + 2.0 ** -20 * r.abs()


def _ids(gpu, kind, m, pool, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "runs":                        # requests one after the other
        ids = torch.repeat_interleave(torch.randint(-1, pool, (m,), generator=g), torch.randint(1, 90, (m,), generator=g))[:m]
    elif kind == "mixed":
        ids = torch.randint(-2, pool + 2, (m,), generator=g)
    elif kind == "one":
        ids = torch.full((m,), pool - 1)
    else:
        ids = torch.full((m,), -1)
    return ids.to(torch.int32).to(gpu)


# (k, widths, paired, rank, pool, rows, ids)
CASES = [
    (32, [16], False, 1, 1, 1, "one"),
    (128, [16], False, 8, 3, 5, "mixed"),
    (1024, [2048, 1024, 1024], False, 16, 32, 16, "mixed"),
    (1024, [128, 256, 128], False, 20, 4, 70, "runs"),
    (256, [128, 128, 128, 128], False, 64, 5, 257, "mixed"),
    (2048, [1024], False, 128, 2, 33, "one"),
    (160, [272], False, 33, 7, 300, "runs"),
    (1024, [48], False, 256, 3, 66, "mixed"),
    (512, [96], True, 16, 4, 40, "mixed"),
    (1024, [6144], True, 8, 16, 9, "runs"),
    (352, [80], True, 100, 2, 513, "runs"),
    (6144, [2048], False, 32, 8, 701, "runs"),
    (128, [64], False, 4, 511, 3000, "mixed"),
    (128, [64], False, 4, 2, 4097, "runs"),
    (64, [32], False, 4, 3, 130, "none"),
]


@pytest.mark.parametrize("k,widths,paired,rank,pool,m,kind", CASES, ids=[f"{c[0]}-{'_'.join(map(str, c[1]))}-r{c[3]}-m{c[5]}-{c[6]}" for c in CASES])
def test_adapter_add(gpu, k, widths, paired, rank, pool, m, kind):
    g, a, b, scales, pool_ = _make(gpu, k, widths, paired, rank, pool)
    ids = _ids(gpu, kind, m, pool)
    x = torch.randn(m, k, device=gpu, generator=g).to(BF16)
    y = torch.randn(m, sum(widths), device=gpu, generator=g).to(BF16)
    plan = ops.AdapterPlan(ids, pool)
    ref, err = _reference(y, x, a, b, scales, widths, paired, ids)
    out = ops.adapter_add(y, x, pool_, plan, out=torch.full_like(y, NAN))
    _check(out, ref, err)
    none = (ids < 0) | (ids >= pool)
    assert torch.equal(out[none], y[none])
    if paired:
        act = ops.adapter_add(y, x, pool_, plan, swiglu=True)
        _check(act, *_swiglu(ref, err))
        assert act.shape == (m, sum(widths) // 2)
    again = ops.adapter_add(y, x, pool_, plan, workspace=ops.Workspace())
    assert again is y and torch.equal(y, out), "in place"


def test_plan_keeps_every_row_once(gpu):
    for m, pool, kind in ((1, 1, "one"), (1000, 7, "mixed"), (5000, 511, "mixed"), (70000, 3, "runs"), (64, 1, "none")):
        ids = _ids(gpu, kind, m, pool, seed=m)
        plan = ops.AdapterPlan(ids, pool)
        cap = m // 64 + min(pool + 1, m)
        tiles, i = plan.table.view(cap, 68).cpu().tolist(), ids.cpu().long()
        i = torch.where((i < 0) | (i >= pool), pool, i)
        order, at = [], 0
        for a, first, rows, _, *places in tiles:
            if rows:
                assert first == at and rows <= 64
                order += places[:rows]
                assert all(int(i[r]) == (a if a >= 0 else pool) for r in places[:rows])
                at += rows
        assert order == torch.sort(i, stable=True).indices.tolist()
        assert at == m


def test_rows_do_not_touch_each_other(gpu):
    """NaN and infinities in one row's x stay in that row; padding ranks do not make NaN of an infinity."""
    k, pool, rank = 256, 3, 20
    g, a, b, scales, pool_ = _make(gpu, k, [128], False, rank, pool)
    ids = torch.tensor([0, 1, 1, -1, 0, 2, 2, 2], dtype=torch.int32, device=gpu)
    x = torch.randn(8, k, device=gpu, generator=g).to(BF16)
    y = torch.randn(8, 128, device=gpu, generator=g).to(BF16)
    plan = ops.AdapterPlan(ids, pool)
    clean = ops.adapter_add(y, x, pool_, plan, out=torch.empty_like(y))
    for bad in (NAN, float("inf")):
        z = x.clone()
        z[[2, 3, 6], 17] = bad
        got = ops.adapter_add(y, z, pool_, plan, out=torch.empty_like(y))
        keep = torch.tensor([0, 1, 3, 4, 5, 7], device=gpu)
        assert torch.equal(got[keep], clean[keep])
        assert not torch.isfinite(got[[2, 6]].float()).any()
    # an infinity times one rank alone: signed infinities, as the definition has
    one = ops.Adapters(torch.ones(1, 1, 32, dtype=BF16, device=gpu), torch.tensor([1.0, -1.0] * 8, device=gpu).to(BF16).view(1, 16, 1))
    z = torch.zeros(1, 32, dtype=BF16, device=gpu)
    z[0, 5] = float("inf")
    got = ops.adapter_add(torch.zeros(1, 16, dtype=BF16, device=gpu), z, one, ops.AdapterPlan(torch.zeros(1, dtype=torch.int32, device=gpu), 1))
    assert got[0].tolist() == [float("inf"), float("-inf")] * 8


def test_put(gpu):
    g, a, b, scales, pool_ = _make(gpu, 128, [128, 128], False, 24, 3)
    x, y = torch.randn(6, 128, device=gpu, generator=g).to(BF16), torch.randn(6, 256, device=gpu, generator=g).to(BF16)
    ids = torch.tensor([0, 1, 2, 1, -1, 1], dtype=torch.int32, device=gpu)
    plan = ops.AdapterPlan(ids, 3)
    na, nb = torch.randn(2, 8, 128, device=gpu, generator=g).to(BF16), torch.randn(256, 8, device=gpu, generator=g).to(BF16)
    pool_.put(1, na, nb, 0.5)
    a[1], b[1], scales[1] = 0, 0, 0.5
    a[1, :, :8], b[1, :, :8] = na, nb
    _check(ops.adapter_add(y, x, pool_, plan, out=torch.empty_like(y)), *_reference(y, x, a, b, scales, [128, 128], False, ids))
    for args in ((3, na, nb), (-1, na, nb), (1, na[0], nb), (1, na, nb[:, :4]), (1, na.float(), nb), (1, na[:, :, :64], nb)):
        with pytest.raises(ValueError):
            pool_.put(*args)


def test_pools_past_32_bit_offsets(gpu):
    """b of over 4 GB: its last adapters."""
    n, rank, k, pool = 16384, 256, 64, 511
    b = torch.zeros(pool, n, rank, dtype=BF16, device=gpu)
    a = torch.zeros(pool, 1, rank, k, dtype=BF16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    a[-1], b[-1] = torch.randn(rank, k, device=gpu, generator=g).to(BF16), torch.randn(n, rank, device=gpu, generator=g).to(BF16)
    scales = torch.ones(pool, device=gpu)
    pool_ = ops.Adapters(a, b, scales)
    x, y = torch.randn(3, k, device=gpu, generator=g).to(BF16), torch.zeros(3, n, dtype=BF16, device=gpu)
    ids = torch.tensor([pool - 1, 0, pool - 1], dtype=torch.int32, device=gpu)
    ref, err = _reference(y, x, a, b, scales, [n], False, ids)
    _check(ops.adapter_add(y, x, pool_, ops.AdapterPlan(ids, pool)), ref, err)


def test_captured_and_replayed(gpu):
    g, a, b, scales, pool_ = _make(gpu, 256, [192], True, 16, 6)
    m = 90
    x, y = torch.randn(m, 256, device=gpu, generator=g).to(BF16), torch.randn(m, 192, device=gpu, generator=g).to(BF16)
    ids, ws = _ids(gpu, "runs", m, 6), ops.Workspace()
    plan, act = ops.AdapterPlan(ids, 6), torch.empty(m, 96, dtype=BF16, device=gpu)

    def step(plan, act, w=None):
        plan.refresh()
        ops.adapter_add(y, x, pool_, plan, out=act, swiglu=True, workspace=w)

    step(plan, act, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(plan, act, ws)
    other, want = ops.AdapterPlan(ids, 6), torch.empty_like(act)
    for i, kind in enumerate(("mixed", "none", "one", "runs")):
        ids.copy_(_ids(gpu, kind, m, 6, seed=i))
        x.copy_(torch.randn(m, 256, device=gpu, generator=g))
        pool_.put(2, a[5], b[5] * i, 0.3)
        graph.replay()
        step(other, want)
        torch.cuda.synchronize()
        assert torch.equal(act, want)


def test_another_stream(gpu):
    g, a, b, scales, pool_ = _make(gpu, 256, [128], False, 16, 4)
    x, y = torch.randn(40, 256, device=gpu, generator=g).to(BF16), torch.randn(40, 128, device=gpu, generator=g).to(BF16)
    ids = _ids(gpu, "mixed", 40, 4)
    plan = ops.AdapterPlan(ids, 4)
    want = ops.adapter_add(y, x, pool_, plan, out=torch.empty_like(y))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = [ops.adapter_add(y, x, pool_, p, out=torch.empty_like(y)) for p in (plan, ops.AdapterPlan(ids, 4))]
    other.synchronize()
    assert all(torch.equal(o, want) for o in got)


def test_no_rows(gpu):
    _, _, _, _, pool_ = _make(gpu, 64, [32], True, 4, 2)
    plan = ops.AdapterPlan(torch.zeros(0, dtype=torch.int32, device=gpu), 2)
    y, x = torch.zeros(0, 32, dtype=BF16, device=gpu), torch.zeros(0, 64, dtype=BF16, device=gpu)
    assert ops.adapter_add(y, x, pool_, plan) is y and ops.adapter_add(y, x, pool_, plan, swiglu=True).shape == (0, 16)


def test_refusals(gpu):
    g, a, b, scales, pool_ = _make(gpu, 128, [128, 128], False, 8, 3)
    x, y = torch.zeros(5, 128, dtype=BF16, device=gpu), torch.zeros(5, 256, dtype=BF16, device=gpu)
    ids = torch.zeros(5, dtype=torch.int32, device=gpu)
    plan = ops.AdapterPlan(ids, 3)
    make = lambda **kw: ops.Adapters(**{**dict(a=a, b=b, scales=scales, widths=[128, 128]), **kw})  # noqa: E731
    make()
    for kw in (dict(a=a.float()), dict(a=a.cpu()), dict(a=a[:2]), dict(a=a[0]), dict(b=b[:, :, :4].contiguous()), dict(widths=None),
               dict(widths=[64, 192]), dict(widths=[128, 256]), dict(widths=[128.0, 128]), dict(paired=True), dict(scales=scales[:2]),
               dict(scales=scales.double()), dict(a=a[..., :100].contiguous()), dict(b=b[:, :248].contiguous(), widths=[128, 120])):
        with pytest.raises(ValueError):
            make(**kw)
    wide = torch.zeros(1, 32, 64, dtype=BF16, device=gpu)
    for rank, pool in ((257, 1), (4, 512)):
        with pytest.raises(ValueError):
            ops.Adapters(torch.zeros(pool, rank, 32, dtype=BF16, device=gpu), torch.zeros(pool, 16, rank, dtype=BF16, device=gpu))
    assert wide is not None
    for args in ((ids.long(), 3), (ids.cpu(), 3), (ids, 0), (ids, 512), (ids, 2.5), (ids.view(1, 5), 3)):
        with pytest.raises(ValueError):
            ops.AdapterPlan(*args)
    for kw in (dict(y=y[:4]), dict(x=x[:, :64].contiguous()), dict(x=x.float()), dict(plan=ops.AdapterPlan(ids, 4)), dict(swiglu=True),
               dict(out=torch.empty(5, 128, dtype=BF16, device=gpu)), dict(out=torch.empty(5, 256, device=gpu)), dict(y=y.T),
               dict(adapters=None), dict(plan=None)):
        with pytest.raises(ValueError):
            ops.adapter_add(**{**dict(y=y, x=x, adapters=pool_, plan=plan), **kw})
    pair = ops.Adapters(a, b, scales, paired=True)
    with pytest.raises(ValueError, match="must not be y|out must be"):
        ops.adapter_add(y, x, pair, plan, out=y, swiglu=True)


def test_out_may_be_x(gpu):
    """x is done with when the first result is written."""
    g = torch.Generator(device=gpu).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device=gpu, generator=g).to(torch.bfloat16)  # noqa: E731
    for m in (3, 700):
        x, y = rnd(m, 256), rnd(m, 256)
        pool = ops.Adapters(rnd(3, 8, 256), rnd(3, 256, 8))
        plan = ops.AdapterPlan((torch.arange(m, device=gpu) % 4).to(torch.int32), 3)
        want = ops.adapter_add(y, x, pool, plan, out=torch.empty_like(y))
        got = ops.adapter_add(y, x, pool, plan, out=x)
        assert got is x and torch.equal(got, want)


@pytest.mark.parametrize("paired", [False, True])
def test_rows_without_an_adapter_keep_their_bits(gpu, paired):
    """Every bf16 pattern there is, negative zeros and NaN among them, into another tensor and in place."""
    y = torch.arange(65536, device=gpu).to(torch.int16).view(BF16).view(256, 256)
    g, a, b, scales, pool = _make(gpu, 64, [256] if paired else [128, 128], paired, 8, 2)
    x = torch.randn(256, 64, device=gpu, generator=g).to(BF16)
    ids = torch.full((256,), -1, dtype=torch.int32, device=gpu)
    ids[200:203] = 1                                       # others among them
    plan, none = ops.AdapterPlan(ids, 2), ids < 0
    out = ops.adapter_add(y, x, pool, plan, out=torch.zeros_like(y))
    assert torch.equal(out.view(torch.int16)[none], y.view(torch.int16)[none])
    keep = y.clone()
    ops.adapter_add(y, x, pool, plan)
    assert torch.equal(y.view(torch.int16)[none], keep.view(torch.int16)[none])


def test_more_slices_than_four(gpu):
    g = torch.Generator(device=gpu).manual_seed(6)
    rnd = lambda *s: torch.randn(*s, device=gpu, generator=g).to(BF16)  # noqa: E731
    ops.Adapters(rnd(1, 4, 8, 64), rnd(1, 512, 8), widths=[128] * 4)
    with pytest.raises(ValueError, match="slices"):
        ops.Adapters(rnd(1, 5, 8, 64), rnd(1, 640, 8), widths=[128] * 5)
