"""Sizes past what a launch or a 32-bit argument holds are refused before anything is launched."""

import pytest
import torch

from torch2iron_amd import _lib, ops

FAKE = 0x10000          # an aligned, never-dereferenced address
E = _lib


def test_entry_points_refuse_grids_past_32_bits():
    """A launch has fewer than 2^32 threads: 2^24 workgroups of 256 are too many."""
    lib = _lib.load()
    many = 2 ** 24

    def packed_prep(rows):
        return lib.t2i_packed_qk_rope_kv(FAKE, rows, FAKE, FAKE, 2, 16, 8, 128, FAKE, FAKE, 1e-6, FAKE, 0, FAKE, FAKE, FAKE, 64, None)

    def packed_attn(n_bins, n_merges):
        nbytes = lib.t2i_packed_attention_workspace_bytes(2, 8)
        return lib.t2i_packed_attention(FAKE, 5, FAKE, 3, FAKE, n_merges, 2, FAKE, n_bins, 16, 8, 128, FAKE, FAKE, 2, 64, FAKE,
                                        None, FAKE, nbytes, None)

    def tree_prep(b):
        return lib.t2i_tree_qk_rope_kv(FAKE, FAKE, FAKE, None, b, 64, 16, 8, 128, FAKE, FAKE, 1e-6, FAKE, 0, FAKE, FAKE, FAKE, 64, None)

    def tree_attn(b):
        nbytes = lib.t2i_tree_attention_workspace_bytes(b, 64, 1024, 64, 64)
        return lib.t2i_tree_attention(FAKE, FAKE, FAKE, None, b, 64, 1024, 64, 128, FAKE, FAKE, 64, FAKE, FAKE, nbytes, None)

    def commit(layers):
        return lib.t2i_tree_commit(FAKE, FAKE, FAKE, FAKE, None, layers, 64, 8, 64, 128, FAKE, FAKE, 64, FAKE, FAKE, FAKE, FAKE + 4096, None)

    def logprobs(m, v):
        return lib.t2i_token_logprobs(FAKE, 0, v, m, v, FAKE, 0, FAKE, FAKE, None, None, None, 0, None)

    assert packed_prep(many) == E.T2I_ERR_SHAPE
    assert packed_attn(many // 8, 1) == E.T2I_ERR_SHAPE and packed_attn(3, many // 8) == E.T2I_ERR_SHAPE
    assert tree_prep(many // 64) == E.T2I_ERR_SHAPE and tree_attn(many // 64 // 128) == E.T2I_ERR_SHAPE
    assert commit(4 * many // 64 // 64) == E.T2I_ERR_SHAPE
    assert logprobs(many, 8) == E.T2I_ERR_SHAPE


@pytest.mark.gpu
def test_logits_past_32_bit_sizes_are_refused(gpu):
    """2^32 + 8 logits a row are not 8; nothing is read, so nothing need be written first."""
    wide = torch.empty(1, 2 ** 32 + 8, dtype=torch.float16, device=gpu)
    with pytest.raises(ValueError, match="too many"):
        ops.token_logprobs(wide, torch.zeros(1, dtype=torch.int32, device=gpu))
