"""Rows of log probabilities with many NaN: their places, and what they cost."""

import pytest
import torch

from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _ranked(x, k):
    """NaN first, then larger values, the lower index first among equals."""
    key = torch.where(x.isnan(), torch.full_like(x, float("inf")), x.clamp(max=torch.finfo(x.dtype).max))
    return torch.sort(key + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v,k,offset", [(40, 32, 0), (3001, 5, 3), (20011, 20, 1), (151936, 8, 0)])
def test_places_of_nan(gpu, dtype, v, k, offset):
    """As many NaN as alternatives, one fewer, one more, and everywhere, over every part, the ends of a row that
    no 16-byte piece holds, and rows in one piece."""
    g = torch.Generator(device=gpu).manual_seed(v + k)
    for copies in (1, 150):
        x = (torch.randn(9, v + offset, device=gpu, generator=g) * 2).to(dtype)
        for row, n in enumerate((k - 1, k, k + 1, 3 * k)):
            x[row, offset + torch.randperm(v, device=gpu, generator=g)[:n]] = NAN
        x[4] = NAN
        x[5, offset:offset + v // 2] = NAN
        x[6, offset + v // 2:] = NAN
        x[7, offset + v - k:] = NAN
        x = x.repeat(copies, 1)[:, offset:]
        t = torch.zeros(x.shape[0], dtype=torch.int32, device=gpu)
        lp, ent, top, ids = ops.token_logprobs(x, t, top_k=k)
        assert torch.equal(ids.long(), _ranked(x, k))
        odd = torch.arange(x.shape[0], device=gpu) % 9 < 8
        odd &= x.isnan().any(-1)
        assert lp[odd].isnan().all() and ent[odd].isnan().all() and top[odd].isnan().all()
        assert torch.isfinite(lp[8::9]).all() and torch.isfinite(ent[8::9]).all() and torch.isfinite(top[8::9]).all()


def _time(f, n=5):
    f()
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(n + 1)]
    ev[0].record()
    for e in ev[1:]:
        f()
        e.record()
    torch.cuda.synchronize()
    return sorted(a.elapsed_time(b) for a, b in zip(ev, ev[1:]))[n // 2]


def test_cost_of_rows_of_nan(gpu):
    """A list of NaN lets no later value in: rows of nothing else cost what other rows do."""
    x = torch.randn(1000, 100003, device=gpu)
    t = torch.zeros(1000, dtype=torch.int32, device=gpu)
    ws = ops.Workspace()
    run = lambda: ops.token_logprobs(x, t, top_k=20, workspace=ws)  # noqa: E731
    usual = _time(run)
    x[:] = NAN
    assert _time(run) <= 3 * usual
