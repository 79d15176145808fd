"""Drafted tokens verified on the MI355X against the definition in float64, row by row on the CPU.

Tokens and counts are whole numbers and must be equal: weights and running sums are float64 on both sides (a weight off
by 1e-13 relative, sums of them no more), so a number u falls between the two sides' borders with a probability of tokens *
2e-13 at most; `_reference` asserts for each case that no number lies within 1e-12 of a border.
Log probabilities: fp32 rounding of a float64 value, 2^-24 relative, and 1e-13 of the float64 terms' size."""

import math

import pytest
import torch

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
NAN = float("nan")
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _reference(logits, starts, tokens, uniforms, probs, temps):
    """counts, next, logprobs; asserts that no decision hangs on a difference below 1e-12 of its sum."""
    x_all = logits.double().cpu()
    tokens, u = tokens.tolist(), uniforms.double().tolist()
    q_all = None if probs is None else probs.double().cpu()
    v = x_all.shape[1]
    counts, nxt, lps = [], [], torch.zeros(x_all.shape[0], dtype=torch.float64)
    ascends = starts == sorted(starts) and starts[0] >= 0 and starts[-1] <= x_all.shape[0]
    for s in range(len(starts) - 1):
        a, e = starts[s], starts[s + 1]
        if a == e or not ascends:
            counts.append(0)
            nxt.append(-1)
            continue
        temp = 1.0 if temps is None else float(temps[s])
        greedy = not temp > 0
        for row in range(a, e):
            x = x_all[row]
            if not torch.isfinite(x.max()) or torch.isnan(x).any():
                counts.append(row - a)
                nxt.append(-1)
                lps[row] = NAN
                break
            y = (x - x.max()) / (1.0 if greedy else temp)
            y = torch.where(x == -math.inf, -math.inf, y)
            p = torch.exp(y)
            z = float(p.sum())
            p = p / z
            best = int((x == x.max()).nonzero()[0])
            last = row == e - 1
            if not last:
                t = tokens[row + 1]
                inside = 0 <= t < v
                q = 1.0 if q_all is None else float(q_all[row, t]) if inside else 0.0
                pt = float(p[t]) if inside else 0.0
                if not greedy:
                    assert abs(u[row] * q - pt) > 1e-12 * pt or not inside or u[row] * q == pt == 0, "too near a border"
                if inside and (t == best if greedy else u[row] * q < pt):
                    lps[row] = float(y[t]) - math.log(z)
                    continue
            w = p.clone()
            if not last:
                if q_all is None:
                    if inside:
                        w[t] = 0
                else:
                    w = (p - q_all[row]).clamp(min=0)
                if not float(w.sum()) > 0:
                    w = p
            c = w.cumsum(0)
            target = u[e - 1] * float(c[-1])
            if not greedy:
                k = int(torch.searchsorted(c, torch.tensor(target, dtype=torch.float64), right=True))
                near = [abs(float(c[i]) - target) for i in (k - 1, k) if 0 <= i < v and w[i] > 0]
                assert u[e - 1] in (0.0, 1.0) or min(near) > 1e-12 * float(c[-1]), "too near a border"
                hits = ((c > target) & (w > 0)).nonzero()
                k = int(hits[0]) if len(hits) else int((w > 0).nonzero()[-1])
            else:
                k = best
            counts.append(row - a)
            nxt.append(k)
            lps[row] = float(y[k]) - math.log(z)
            break
    return counts, nxt, lps


def _case(gpu, lens, v, dtype, with_probs, seed, sharp=1.0, greedy_every=4):
    g = torch.Generator().manual_seed(seed)
    m = sum(lens)
    x = torch.randn(m, v, generator=g) * 2 * sharp
    hot = (torch.randint(0, v, (m, 1), generator=g) + torch.arange(min(v, 5)) * max(1, v // 5)) % v
    x.scatter_(1, hot, 9 + 2 * torch.randn(m, hot.shape[1], generator=g))
    draft = x + 0.8 * torch.randn(m, v, generator=g)
    q = torch.softmax(draft, -1)
    after = torch.multinomial(q, 1, generator=g)[:, 0]
    tokens = after.roll(1).to(torch.int32)
    temps = 0.5 + torch.rand(len(lens), generator=g)
    temps[::greedy_every] = 0.0
    temps[1::2 * greedy_every] = 1.0
    starts = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    u = torch.rand(m, generator=g)
    dev = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    return (x.to(dtype).to(gpu), dev(starts), dev(tokens), dev(u), dev(q) if with_probs else None, dev(temps))


def _check(args, got, near=1e-13):
    logits, starts, tokens, u, probs, temps = args
    counts, nxt, lps = _reference(logits, starts.tolist(), tokens, u, probs, temps)
    assert got[0].tolist() == counts and got[1].tolist() == nxt
    lp = got[2].double().cpu()
    assert torch.equal(torch.isnan(lp), torch.isnan(lps))
    ok = ~torch.isnan(lps)
    err = (lp - lps)[ok].abs()
    # the float64 terms: (x - m) / T up to a few hundred, ln Z up to 12
    assert (err <= 2.0 ** -24 * lps[ok].abs() + near * (lps[ok].abs() + 100)).all(), err.max()


SHAPES = [([1], 5), ([1], 1), ([2], 1), ([3, 1, 4], 7), ([5, 0, 1, 9], 1000), ([4] * 6, 1023), ([2, 6], 1024), ([9, 3], 1025),
          ([5] * 5, 4099), ([1] * 40, 30011), ([17, 2], 2049), ([5, 3, 1], 151936), ([2, 3], 300001),
          ([2, 1], 1100003), ([3, 1] * 150, 1500), ([2, 0, 1] * 700, 65)]


@pytest.mark.parametrize("with_probs", [False, True], ids=["certain", "probs"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,v", SHAPES, ids=[f"{'_'.join(map(str, s[0][:5]))}-{s[1]}" for s in SHAPES])
def test_verify(gpu, lens, v, dtype, with_probs):
    args = _case(gpu, lens, v, TYPES[dtype], with_probs, seed=v + len(lens))
    got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
    again = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5], workspace=ops.Workspace())
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    _check(args, got)


def test_every_outcome_occurs(gpu):
    """Over the cases below drafts are refused at once, in the middle and not at all."""
    seen = set()
    for seed in range(4):
        args = _case(gpu, [4] * 32, 300, torch.float32, True, seed=seed, greedy_every=5)
        got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
        _check(args, got)
        seen |= set(got[0].tolist())
    assert seen == {0, 1, 2, 3}


def test_distribution(gpu):
    """With uniform numbers the token after the row is distributed as p, whatever the draft's distribution: 20000 sequences
    of one draft over 6 tokens against p, within 5 standard deviations of a count."""
    n, v = 20000, 6
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, -math.inf, 1.0], device=gpu)
    q = torch.tensor([0.1, 0.4, 0.1, 0.2, 0.1, 0.1], device=gpu)
    draft = torch.multinomial(q, n, replacement=True, generator=g).to(torch.int32)
    tokens = torch.stack([torch.zeros_like(draft), draft], 1).view(-1).contiguous()
    u = torch.rand(2 * n, device=gpu, generator=g)
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=gpu)
    counts, nxt, _ = ops.verify_drafts(x.expand(2 * n, v).contiguous(), starts, tokens, u, draft_probs=q.expand(2 * n, v).contiguous())
    first = torch.where(counts == 1, draft, nxt)
    p = torch.softmax(x.double(), 0).cpu()
    hist = torch.bincount(first.long().cpu(), minlength=v).double()
    assert ((hist - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1e-9).all(), hist / n


def test_masks_and_rows_without_a_distribution(gpu):
    v = 2100
    for with_probs in (False, True):
        args = list(_case(gpu, [3] * 10, v, torch.float32, with_probs, seed=5, greedy_every=3))
        x = args[0]
        x[:, 100:1200] = -math.inf                        # masked tokens
        x[3, 7] = NAN                                     # sequence 1, its first row
        x[7, v - 1] = math.inf                            # sequence 2, its middle row
        x[9:12] = -math.inf                               # sequence 3
        x[12:15] = torch.finfo(torch.float32).min         # sequence 4: the lowest values, all alike
        x[15:18, 5:] = torch.finfo(torch.float32).min     # sequence 5: as a mask
        x[18:21, 1:] = -math.inf                          # sequence 6: one token
        got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
        _check(args, got)
        assert got[1][1] == -1 and got[1][3] == -1 and got[1][6] == 0


def test_extreme_temperatures_and_numbers(gpu):
    for with_probs in (False, True):
        args = list(_case(gpu, [3] * 12, 500, torch.float32, with_probs, seed=6))
        args[5] = torch.tensor([1e-30, 1e-3, 1e30, math.inf, -1.0, NAN, -0.0, 100.0, 1e-45, 0.01, 3.0, 1.0], device=gpu)
        ref = list(args)
        ref[5] = torch.tensor([0.0 if not t > 0 else t for t in args[5].tolist()], dtype=torch.float64)
        got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
        # lowest positive temperatures: weights of 0 and 1 (the reference in float64 has them too); terms of 1e30 / T stay
        # within 2^-24 of themselves, where they are finite
        counts, nxt, _ = _reference(ref[0], ref[1].tolist(), ref[2], ref[3], ref[4], ref[5])
        assert got[0].tolist() == counts and got[1].tolist() == nxt
        args = list(_case(gpu, [1] * 4, 500, torch.float32, with_probs, seed=7, greedy_every=9))
        args[3] = torch.tensor([0.0, 1.0, 2.0, 1 - 2.0 ** -24], device=gpu)
        _check(args, ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5]))


def test_logits_of_any_size(gpu):
    """Differences are taken before they are scaled: rows far from 0, and of huge values."""
    for with_probs in (False, True):
        for scale, shift in ((1.0, 3e4), (1.0, -2e6), (1e30, 0.0), (1e3, 1e9), (1e-20, 0.0)):
            args = list(_case(gpu, [3, 1, 4], 2500, torch.float32, with_probs, seed=17))
            args[0] = args[0] * scale + shift
            _check(args, ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5]), near=1e-13 * max(1.0, scale))


def test_nothing_left_of_the_rest(gpu):
    """q at or above p everywhere (or the draft certain) and yet refused, by a number of 1: the token comes from p."""
    x = torch.tensor([[-math.inf, 4.0, -math.inf, 2.0]] * 2 + [[-math.inf, 4.0, -math.inf, -math.inf]] * 2, device=gpu)
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device=gpu)
    tokens = torch.tensor([0, 1, 0, 1], dtype=torch.int32, device=gpu)
    q = torch.tensor([[0.0, 1.0, 0.0, 1.0]] * 4, device=gpu)
    for u in ([1.0, 0.5, 1.0, 0.5], [1.0, 0.95, 1.0, 0.0], [NAN, 0.3, NAN, 0.3]):
        u = torch.tensor(u, device=gpu)
        for probs in (q, None):
            counts, nxt, lp = ops.verify_drafts(x, starts, tokens, u, draft_probs=probs)
            # certain draft: token 3 is what is left in the first sequence, nothing in the second
            first = 3 if probs is None else 3 if u[1] > 0.9 else 1
            assert counts.tolist() == [0, 0] and nxt.tolist() == [first, 1]
            assert torch.isfinite(lp).all()


def test_equal_maxima(gpu):
    """Greedy: the lowest index, over the borders of chunks, among both zeros."""
    v = 5000
    x = torch.full((4, v), -1.0, device=gpu)
    x[0, [4999, 1024, 1023]] = 2.0
    x[1, [3000, 2999]] = 2.0
    x[2, 4000], x[2, 700] = 0.0, -0.0
    x[3] = 0.5
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device=gpu)
    tokens = torch.tensor([9, 1023, 9, 700], dtype=torch.int32, device=gpu)
    counts, nxt, _ = ops.verify_drafts(x, starts, tokens, torch.rand(4, device=gpu), temperatures=torch.zeros(2, device=gpu))
    assert counts.tolist() == [1, 1] and nxt.tolist() == [2999, 0]
    tokens[1], tokens[3] = 1024, 4000                      # another of the largest is not the first
    counts, nxt, _ = ops.verify_drafts(x, starts, tokens, torch.rand(4, device=gpu), temperatures=torch.zeros(2, device=gpu))
    assert counts.tolist() == [0, 0] and nxt.tolist() == [1023, 700]


def test_drafts_that_are_no_tokens(gpu):
    for with_probs in (False, True):
        args = _case(gpu, [3, 3, 3, 3], 800, torch.float32, with_probs, seed=8, greedy_every=2)
        args[2][[1, 4, 7, 10]] = torch.tensor([-1, 800, 2**31 - 1, -2**31], dtype=torch.int32, device=gpu)
        got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
        _check(args, got)
        assert got[0].tolist() == [0] * 4


def test_row_starts(gpu):
    """Rows of nobody have log probability 0; row_starts that do not ascend within the batch leave no sequence any rows."""
    for starts in ([2, 4, 4, 7], [0, 5, 3, 10], [-1, 3, 6, 10], [0, 3, 11, 10], [10, 10, 10, 10]):
        for with_probs in (False, True):
            args = list(_case(gpu, [10], 300, torch.float32, with_probs, seed=9))
            args[1] = torch.tensor(starts, dtype=torch.int32, device=gpu)
            args[5] = None
            got = ops.verify_drafts(*args[:4], draft_probs=args[4])
            _check(args, got)


def test_strided_and_unaligned_rows(gpu):
    for dtype, v in ((torch.bfloat16, 1031), (torch.float16, 1024), (torch.float32, 2050)):
        args = list(_case(gpu, [4, 2, 5], v, dtype, True, seed=11))
        want = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
        for off in (1, 3):
            wide = torch.full((11, v + 9), NAN, dtype=dtype, device=gpu)
            wide[:, off:off + v] = args[0]
            q = torch.full((11, v + 5), NAN, device=gpu)
            q[:, off:off + v] = args[4]
            q = q[:, off:off + v]
            q[[3, 5, 10]] = NAN                            # behind last rows nothing is drafted
            got = ops.verify_drafts(wide[:, off:off + v], *args[1:4], draft_probs=q, temperatures=args[5])
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_logits_past_32_bit_offsets(gpu):
    """Rows that start past 4 GB."""
    v, m = 151936, 14200
    big = torch.zeros(m, v, dtype=torch.bfloat16, device=gpu)
    args = _case(gpu, [3, 2], v, torch.bfloat16, False, seed=12)
    big[m - 5:] = args[0]
    starts = torch.tensor([0, m - 5, m - 2, m], dtype=torch.int32, device=gpu)
    tokens, u = torch.zeros(m, dtype=torch.int32, device=gpu), torch.full((m,), 0.999, device=gpu)
    tokens[m - 5:], u[m - 5:] = args[2], args[3]
    got = ops.verify_drafts(big, starts, tokens, u, temperatures=torch.cat([torch.ones(1, device=gpu), args[5]]))
    want = ops.verify_drafts(*args[:4], temperatures=args[5])
    assert torch.equal(got[0][1:], want[0]) and torch.equal(got[1][1:], want[1]) and torch.equal(got[2][m - 5:], want[2])


@pytest.mark.parametrize("with_probs", [False, True], ids=["certain", "probs"])
def test_captured_and_replayed(gpu, with_probs):
    args = list(_case(gpu, [5, 1, 3, 6], 4099, torch.bfloat16, with_probs, seed=13))
    ws = ops.Workspace()
    call = lambda w=None: ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5], workspace=w)  # noqa: E731
    call(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(ws)
    for seed in range(4):
        fresh = _case(gpu, [[5, 1, 3, 6], [1, 1, 12, 1], [0, 15, 0, 0], [4, 4, 4, 3]][seed], 4099, torch.bfloat16, with_probs, seed=20 + seed)
        for a, b in zip(args, fresh):
            if a is not None:
                a.copy_(b)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        _check(args, got)


def test_another_stream(gpu):
    args = _case(gpu, [5, 1, 3], 3000, torch.float32, True, seed=14)
    want = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(gpu):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    counts, nxt, lp = ops.verify_drafts(torch.zeros(0, 9, device=gpu), i32(0, 0, 0), i32(), torch.zeros(0, device=gpu))
    assert counts.tolist() == [0, 0] and nxt.tolist() == [-1, -1] and lp.numel() == 0


def test_refusals(gpu):
    x, starts, tokens, u, q, t = _case(gpu, [3, 2], 40, torch.float32, True, seed=15)
    bad = [dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.T), dict(row_starts=starts.long()),
           dict(row_starts=starts[:1]), dict(tokens=tokens[:-1]), dict(tokens=tokens.long()), dict(uniforms=u.double()),
           dict(uniforms=u[1:]), dict(draft_probs=q.bfloat16()), dict(draft_probs=q[:, 1:]), dict(draft_probs=q.cpu()),
           dict(draft_probs=q.T.contiguous().T), dict(temperatures=t[:1]), dict(temperatures=t.double())]
    good = dict(logits=x, row_starts=starts, tokens=tokens, uniforms=u, draft_probs=q, temperatures=t)
    ops.verify_drafts(**good)
    for kw in bad:
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**good, **kw})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,v", [([2] * 140, 30011), ([4] * 140, 30011), ([5, 1, 0, 3] * 7, 151936), ([2, 9] * 9, 300001)],
                         ids=["140x2", "140x4", "28-151936", "18-300001"])
def test_many_sequences_of_many_chunks(gpu, lens, v, dtype):
    """Draft probabilities, the rest of a refused draft's row over several workgroups, and, for rows times chunks of 16384
    and more, two chunks a wave of the rows' pass."""
    args = _case(gpu, lens, v, TYPES[dtype], True, seed=v + len(lens))
    chunks, drafted = -(-v // 1024), sum(n > 1 for n in lens)
    assert len(lens) * -(-chunks // 16) > 256, "decided and summed in one launch"
    got = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5])
    again = ops.verify_drafts(*args[:4], draft_probs=args[4], temperatures=args[5], workspace=ops.Workspace())
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    _check(args, got)
    refused = (got[0].cpu() < torch.tensor(lens) - 1) & (args[5].cpu() > 0)
    assert int(refused.sum()) > drafted // 20, "hardly a draft was refused"
