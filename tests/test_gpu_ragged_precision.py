"""Drafted trees and single rows against float64 to the precision of their decode steps.

Tolerance, elementwise: the output's rounding to bf16 is at most 2^-8 |out|.  A weight is multiplied as two
bf16 words, the second of which is rounded: 2^-8 2^-8 = 2^-16 of the weight.  A score is 128 products
summed in fp32, off by at most 128 2^-24 sum |q k| / sqrt(D) (about 7 in the mean of normal q and k, 11
at the most here): 9e-5, and so is its weight, twice over with the normaliser's.  fp32 sums over up to
4100 keys: 4100 2^-24 = 2.5e-4 of sum p |v| at the very worst.  Together below 2^-11 (sum p |v| + |out|)."""

import pytest
import torch
from test_gpu_ragged import _packed_case, _packed_reference, _tree_case, _tree_reference

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu


def _check(out, ref, mag, what=""):
    err = (out.double() - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -11 * (mag + ref.abs())
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()}, worst {(err - tol).max():.3e} over"


@pytest.mark.parametrize("hq,hkv,cap,ctx,n,counts", [
    (16, 8, 128, [0, 3, 40], 8, None), (2, 1, 200, [63, 64, 65], 8, [8, 1, 5]), (8, 1, 300, [20, 60], 37, None),
    (32, 8, 400, [30, 200, 7], 64, [64, 64, 9]), (32, 4, 400, [0, 129], 64, None), (4, 1, 4000, [3000], 20, None)])
def test_tree_attention(gpu, hq, hkv, cap, ctx, n, counts):
    q, parents, ctx_t, counts_t, kc, vc, counts_l = _tree_case(gpu, hq, hkv, cap, ctx, n, counts, "random")
    ref, mag = _tree_reference(q, parents, ctx, counts_l, kc, vc, cap)
    out = ops.tree_attention(q, parents, ctx_t, hkv, kc, vc, node_counts=counts_t).view(ref.shape)
    for i, c in enumerate(counts_l):
        _check(out[i, :c], ref[i, :c], mag[i, :c], f"sequence {i}")


@pytest.mark.parametrize("hq,hkv,cap,lengths,starts", [
    (16, 8, 320, [1, 1, 1, 1], [0, 5, 63, 300]), (32, 8, 700, [1, 65, 1, 130, 1], [12, 0, 640, 300, 64]),
    (40, 1, 100, [1, 1], [30, 99]), (200, 1, 90, [1], [70]), (4, 1, 4000, [1, 1], [3999, 2000])])
def test_single_rows(gpu, hq, hkv, cap, lengths, starts):
    """A sequence of one row is a decode step, alone or among chunks of prompts."""
    plan, q, kc, vc = _packed_case(gpu, hq, hkv, cap, lengths, starts, None, len(lengths))
    ref, mag = _packed_reference(plan, q, kc, vc)
    out = ops.packed_attention(q, plan, kc, vc)
    for s, n in enumerate(lengths):
        if n == 1:
            r = plan.first_rows[s]
            _check(out[r], ref[r], mag[r], f"sequence {s}")


def test_single_row_of_equal_values_is_exact(gpu):
    """Constant values come back bit for bit: 1.375 by weights that sum to 1 within a few 2^-16."""
    plan, q, kc, vc = _packed_case(gpu, 8, 2, 700, [1, 1], [20, 650], None, 2)
    vc[:] = 1.375
    assert (ops.packed_attention(q, plan, kc, vc) == 1.375).all()
