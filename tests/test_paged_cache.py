"""The page table's host side and a step's layout; CPU only."""

import pytest
import torch

from torch2iron_amd import model as gm

CFG = gm.Qwen3Config(n_layers=1, hidden=128, n_heads=1, n_kv_heads=1, vocab=32, intermediate=128)


def test_pages_are_given_out_once_and_come_back():
    c = gm.PagedCache(CFG, 3, 10, 8, "cpu", page_slots=16)
    c.reserve(0, 1)
    c.reserve(1, 33)
    c.reserve(0, 16)
    c.reserve(0, 17)
    c.reserve(2, 0)
    used = c.table[c.table >= 0].tolist()
    assert len(used) == len(set(used)) == 5 and c.free_pages == 5
    assert (c.table[0, 2:] == -1).all() and (c.table[1, 3:] == -1).all() and (c.table[2] == -1).all()
    with pytest.raises(RuntimeError, match="free"):
        c.reserve(2, 6 * 16)
    assert c.free_pages == 5 and (c.table[2] == -1).all()
    c.lens[1] = 33
    c.release(1)
    assert c.free_pages == 8 and c.lens[1] == 0 and (c.table[1] == -1).all()
    c.reserve(2, 6 * 16)
    used = c.table[c.table >= 0].tolist()
    assert len(used) == len(set(used)) == 8
    for bad in ((3, 1), (-1, 1), (0, -1), (0, 8 * 16 + 1)):
        with pytest.raises(ValueError):
            c.reserve(*bad)
    for bad in (3, -1):
        with pytest.raises(ValueError):
            c.release(bad)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            gm.PagedCache(CFG, *bad, "cpu")


def test_batch_layout():
    b = gm.PagedBatch([3, 0, 1, 5], [2, 0, 0, 1], device="cpu")
    assert (b.rows, b.n_seqs) == (9, 4)
    assert b.row_starts.tolist() == [0, 3, 3, 4, 9] and b.row_seq.tolist() == [0, 0, 0, 2, 3, 3, 3, 3, 3]
    assert b.head_rows.tolist() == [0, 1, 2, 3, 7, 8] and b.head_starts.tolist() == [0, 3, 3, 4, 6]
    assert b.fed.tolist() == [1, 0, 1, 4]
    assert gm.PagedBatch([2, 1], device="cpu").head_rows.tolist() == [1, 2]
    assert all(t.dtype == torch.int32 for t in (b.row_starts, b.head_rows, b.head_starts, b.fed))


@pytest.mark.parametrize("rows,drafts", [([], None), ([2], [2]), ([0], [1]), ([-1], None), ([2, 3], [1]), ([2.5], None), ([2], [-1])])
def test_batch_refusals(rows, drafts):
    with pytest.raises(ValueError):
        gm.PagedBatch(rows, drafts, device="cpu")
