"""Token log probabilities, entropy and top alternatives on the MI355X against float64.

Tolerance: fp32 logits enter exactly; with u = 2^-24 the sum of up to 2^18 weights is built from
per-lane runs of at most 2400 and a tree, each weight off by a few u from its exponent's fma
(|x - m| log2 e <= 2^7 here: 2^7 u) and v_exp_f32 (one ulp), so log Z and the entropy's mean of
(x - m) are off by at most about (2400 + 130 + 20) u ~ 1.6e-4 of themselves in the worst case and
the square root of the run's length in practice; asserted at 2e-5 of 1 + |value| (x - m, log Z and the
differences of a log probability are at most a few tens, each rounded once: 40 u = 2.4e-6)."""

import math

import pytest
import torch

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _reference(x, tokens, k):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    t = tokens.long()
    ok = (t >= 0) & (t < x.shape[1])
    at = lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    ent = -torch.where(lp == -INF, torch.zeros_like(lp), lp.exp() * lp).sum(-1)
    # stable: equal values (both zeros alike) keep their order
    order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    return torch.where(ok, at, torch.zeros_like(at)), ent, lp.gather(1, order), order


def _check(got, ref):
    for name, g, r in zip(("logprobs", "entropy", "top"), got, ref):
        g = g.double()
        assert torch.equal(g.isnan(), r.isnan()), name
        same = (g == r) | r.isnan()
        err = torch.where(same, torch.zeros_like(r), (g - r).abs() / (1 + r.abs()))
        assert (err <= 2e-5).all(), f"{name}: {err.max():.3e}"
    assert torch.equal(got[3].long(), ref[3]), "ids"


@pytest.mark.parametrize("m,v,k,dtype", [
    (1, 151936, 5, torch.float32), (1, 151936, 32, torch.bfloat16), (3, 1, 1, torch.float32), (2, 2, 2, torch.float16),
    (5, 33, 32, torch.float32), (7, 4097, 8, torch.bfloat16), (64, 4096, 20, torch.float32), (9, 32003, 0, torch.float16),
    (1500, 1001, 3, torch.float32), (13, 151936, 20, torch.float32), (300, 50021, 10, torch.float16), (2, 63, 31, torch.bfloat16)])
def test_random_rows(gpu, m, v, k, dtype):
    g = torch.Generator(device=gpu).manual_seed(m + v + k)
    x = (torch.randn(m, v, device=gpu, generator=g) * 3).to(dtype)
    t = torch.randint(-1, v + 1, (m,), device=gpu, generator=g, dtype=torch.int32)
    got = ops.token_logprobs(x, t, top_k=k)
    _check(got, _reference(x, t, k))
    again = ops.token_logprobs(x, t, top_k=k, workspace=ops.Workspace())
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
def test_strided_rows_from_any_address(gpu, dtype, offset):
    """Rows of a wider array, from an odd column on: no 16-byte boundary in common."""
    m, v, k = 6, 5003, 6
    wide = (torch.randn(m, v + 14, device=gpu, generator=torch.Generator(device=gpu).manual_seed(offset)) * 2).to(dtype)
    wide[:, :offset] = NAN
    wide[:, offset + v:] = NAN
    x = wide[:, offset:offset + v]
    t = torch.tensor([0, 1, v - 1, v // 2, -1, v], dtype=torch.int32, device=gpu)
    _check(ops.token_logprobs(x, t, top_k=k), _reference(x, t, k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v,k", [(40, 32), (3000, 32), (20011, 32), (70003, 7), (9000, 1)])
def test_order_of_equal_values(gpu, v, k, dtype):
    """Equal logits rank by index, both zeros alike, whichever lane, wave or part holds them."""
    x = torch.randint(-2, 3, (40, v), device=gpu, generator=torch.Generator(device=gpu).manual_seed(v)).to(dtype)
    x[8:24] = torch.randn(16, v, device=gpu, generator=torch.Generator(device=gpu).manual_seed(v)).to(torch.bfloat16)
    x[1] = 0.0
    x[1, 1::2] = -0.0
    x[2] = torch.arange(v, device=gpu).float()
    x[3] = -torch.arange(v, device=gpu).float()
    t = torch.zeros(40, dtype=torch.int32, device=gpu)
    _check(ops.token_logprobs(x, t, top_k=k), _reference(x, t, k))
    many = x.repeat(40, 1)                                     # rows in one piece each
    got = ops.token_logprobs(many, t.repeat(40), top_k=k)
    _check([a[-40:] for a in got], _reference(x, t, k))


@pytest.mark.parametrize("v", [50, 9001])
def test_infinite_and_nan_logits(gpu, v):
    """-inf has probability 0; +inf, NaN or nothing but -inf makes a row NaN; other rows are as they are."""
    g = torch.Generator(device=gpu).manual_seed(v)
    x = torch.randn(7, v, device=gpu, generator=g)
    x[1, 3:] = -INF                       # a short list of allowed tokens
    x[2] = -INF
    x[2, v - 1] = 2.5                     # one
    x[3] = -INF                           # none
    x[4, 7] = INF
    x[5, v - 2] = NAN
    x[6] = torch.finfo(torch.float32).min
    x[6, 5] = 1.0
    t = torch.tensor([0, 5, v - 1, 1, 2, 3, 5], dtype=torch.int32, device=gpu)
    lp, ent, top, ids = ops.token_logprobs(x, t, top_k=4)
    rows = [0, 1, 2, 6]
    ref = _reference(x[rows], t[rows], 4)
    _check([a[rows] for a in (lp, ent, top, ids)], ref)
    assert lp[1] == -INF and (ent[2], ent[6]) == (0.0, 0.0)
    assert lp[3:6].isnan().all() and ent[3:6].isnan().all() and top[3:6].isnan().all()
    assert ids[3].tolist() == [0, 1, 2, 3] and ids[4, 0] == 7 and ids[5, 0] == v - 2


def test_masks_of_the_lowest_value(gpu):
    """Rows masked with the type's lowest finite value, some and all of them, and rows at its highest."""
    for dtype in (torch.float32, torch.bfloat16):
        lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
        x = torch.full((4, 5000), lo, device=gpu, dtype=dtype)
        x[1, 77:90] = torch.randn(13, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)).to(dtype)
        x[2] = hi
        x[3, ::2] = hi
        t = torch.tensor([7, 80, 4999, 1], dtype=torch.int32, device=gpu)
        lp, ent, top, ids = ops.token_logprobs(x, t, top_k=5)
        ref = _reference(x[:3], t[:3], 5)
        _check((lp[:3], ent[:3], top[:3], ids[:3]), ref)
        # a difference past fp32's range is a probability of 0
        assert lp[3] == -INF and ids[3].tolist() == [0, 2, 4, 6, 8]
        assert abs(float(ent[3]) - math.log(2500)) < 2e-5 * 9 and (top[3] + math.log(2500)).abs().max() < 2e-5 * 9


def test_large_shift(gpu):
    """A constant added to a row changes nothing but the rounding of its logits."""
    x = torch.randn(3, 30011, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1))
    x = (x + torch.tensor([[0.0], [3e4], [-3e4]], device=gpu))
    t = torch.tensor([5, 6, 7], dtype=torch.int32, device=gpu)
    lp, ent, top, ids = ops.token_logprobs(x, t, top_k=3)
    ref = _reference(x, t, 3)
    for g_, r in zip((lp, ent, top), ref):
        assert ((g_.double() - r).abs() <= 2e-5 * (1 + r.abs())).all()
    assert torch.equal(ids.long(), ref[3])


def test_replayed_from_a_graph(gpu):
    """Split rows and whole rows captured with one workspace; replays follow the inputs."""
    ws = ops.Workspace()
    a, b = torch.randn(2, 60000, device=gpu), torch.randn(2000, 700, device=gpu)
    ta, tb = (torch.zeros(n, dtype=torch.int32, device=gpu) for n in (2, 2000))
    run = lambda: (ops.token_logprobs(a, ta, top_k=4, workspace=ws), ops.token_logprobs(b, tb, top_k=2, workspace=ws))  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = run()
    for i in range(3):
        a.normal_()
        b.normal_()
        ta.random_(0, 60000)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(res, run()):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert math.isfinite(float(res[0][0].sum()))
