"""Softmax weights of 16 bits in the attention over pages, for sequences whose rows times Hq / Hkv are at most 128.

Tolerance, elementwise, of out = sum w_j v_j / sum w_j over n slots, with mag = sum p_j |v_j|.  An addition of a matrix
instruction is off by at most a step, 2^-23 of what is summed (half of it where it rounds), any other by 2^-24.
  scores: 128 products of bf16, exact in fp32: 128 * 2^-23 * A / sqrt(D), A the largest sum |q_d k_d| of a slot; the scale's
    rounding, and the one of its product less the reference: 3 * 2^-24 * S, S the largest score's size; the exponential: 2^-23.
    Together e_w, relative, of a weight: e_w * mag above and e_w * |out| below the line.
  weights: the first bf16 word leaves at most 2^-8 w, the second 2^-8 of that: 2^-16 * mag.
  sums: two products a slot above, one weight below: 2 n 2^-23 * mag + n 2^-24 * |out|.
  parts that are joined, and second-order terms: 2^-20 * mag.
  the output's rounding: 2^-8 * |out|.
Weights rounded to bf16 once would be off by up to 2^-8 * mag instead, and `_once` says for each case that this tolerance tells
the two apart."""

import math

import pytest
import torch

from test_gpu_paged import BF16, CASES, D, Case, _check
from torch2iron_amd import ops

pytestmark = pytest.mark.gpu


def _sequence(c, s):
    """Row range, out, bound, and out from weights that are rounded to bf16 once, of sequence ``s``."""
    at, n, start = sum(c.lens[:s]), c.lens[s], c.ctx[s]
    k, v = (x.double() for x in c.slots[s])
    q, g = c.q[at:at + n].double(), c.hq // c.hkv
    ahead = torch.ones(n, start + n, dtype=torch.bool, device=q.device).triu(start + 1)
    ref, tol, once = (torch.empty(n, c.hq, D, dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(c.hq):
        kh, vh = k[h // g], v[h // g]
        x = ((q[:, h] @ kh.T.contiguous()) / math.sqrt(D)).masked_fill(ahead, -math.inf)
        a = (q[:, h].abs() @ kh.abs().T.contiguous()).masked_fill(ahead, 0.0).amax(-1, keepdim=True)
        size = x.masked_fill(ahead, 0.0).abs().amax(-1, keepdim=True)
        w = torch.exp(x - x.amax(-1, keepdim=True))
        out, mag = (w @ vh) / w.sum(-1, keepdim=True), (w @ vh.abs()) / w.sum(-1, keepdim=True)
        ew = 128 * 2.0 ** -23 * a / math.sqrt(D) + 3 * 2.0 ** -24 * size + 2.0 ** -23
        slots = start + n
        tol[:, h] = (ew + 2.0 ** -16 + 2 * slots * 2.0 ** -23 + 2.0 ** -20) * mag + (ew + slots * 2.0 ** -24 + 2.0 ** -8) * out.abs()
        ref[:, h] = out
        w = w.to(BF16).double()
        once[:, h] = (w @ vh) / w.sum(-1, keepdim=True)
    return slice(at, at + n), ref.view(n, -1), tol.view(n, -1), once.view(n, -1)


def _small(c):
    return [s for s, n in enumerate(c.lens) if 0 < n * (c.hq // c.hkv) <= 128]


def _fine(c, out, tells_apart=True):
    told = False
    for s in _small(c):
        rows, ref, tol, once = _sequence(c, s)
        err = (out[rows].double() - ref).abs()
        assert (err <= tol).all(), f"sequence {s}: worst {(err - tol).max():.3e} over, error {err.max():.3e}"
        told |= bool(((once.to(BF16).double() - ref).abs() > tol).any())
    assert told or not tells_apart


SMALL = [c for c in CASES if any(0 < n * (c[0] // c[1]) <= 128 for n in c[3])]


@pytest.mark.parametrize("hq,hkv,page,lens,ctx", SMALL, ids=[f"{c[0]}-{c[1]}-p{c[2]}-" + "_".join(map(str, c[3][:6])) for c in SMALL])
def test_sequences_of_up_to_128_pairs(gpu, hq, hkv, page, lens, ctx):
    c = Case(gpu, hq, hkv, page, lens, ctx, seed=50)
    # (a single slot has a weight of 1, and the sums' bound for thousands covers what one word leaves of their weights)
    _fine(c, ops.paged_attention(c.q, c.plan, c.k, c.v), any(0 < lens[s] + ctx[s] - 1 < 600 for s in _small(c)))


@pytest.mark.parametrize("lens", [[300, 1, 5, 1, 3, 7, 32], [1, 600, 2, 2, 509]], ids=["one", "two"])
@pytest.mark.parametrize("page", [16, 128])
def test_single_tokens_and_drafts_among_long_chunks(gpu, lens, page):
    ctx = [(1, 40, 12, 0, 31, 250, 17)[i] for i in range(len(lens))]
    c = Case(gpu, 32, 8, page, lens, ctx, seed=51)
    out = ops.paged_attention(c.q, c.plan, c.k, c.v)
    _check(out, *c.reference())
    _fine(c, out)


def test_tiles_that_are_cut(gpu):
    c = Case(gpu, 32, 8, 16, [1, 4, 9], [517, 300, 64], seed=52)
    bins = c.plan.table
    tiles = c.rows * 4 // 128 + 3
    first = bins[8 * tiles:8 * tiles + 4 * max(tiles, 64)].view(-1, 4).cpu()
    assert (first[:, 0] >= 0).sum() > 3, "nothing was cut"
    _fine(c, ops.paged_attention(c.q, c.plan, c.k, c.v))
