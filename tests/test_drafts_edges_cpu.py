"""Drafted tokens: calls at the edge of what is allowed, without a launch (CPU only)."""
import ctypes

import pytest
import torch

from ab_attention import _lib
from ab_attention.streaming import PagedCache, keep_drafts

_A = 4096  # a 16-byte aligned stand-in address: every case is rejected before any runtime call


def _tree_args(**chunk):
    args = _lib.TreeArgs(positions=_A, near=_A, above=_A)
    fields = dict(q=_A, k=_A, v=_A, out=_A, workspace=_A, workspace_bytes=1 << 30, lengths=_A, offsets=_A, page_table=_A, batch=1,
                  heads=2, kv_heads=1, tokens=5, dim=64, pages=3, page_tokens=8, table_width=2, frame=1, scale=0.1,
                  q_stride=(0, 64, 128), k_stride=(512, 512, 64), v_stride=(512, 512, 64), out_stride=(0, 64, 128))
    for name, value in {**fields, **chunk}.items():
        setattr(args.chunk, name, (ctypes.c_int64 * 3)(*value) if isinstance(value, tuple) else value)
    return args


def test_a_tree_has_no_out_rest():
    """What out's rounding takes is not made for a tree, whose split rows are added up by another kernel."""
    lib = _lib.load()
    assert lib.ab_tree_workspace_bytes(ctypes.byref(_tree_args())) > 0
    args = _tree_args(out_rest=_A, workspace=0)  # (without a workspace no launch follows where it is let through)
    assert lib.ab_tree_attention(ctypes.byref(args), None) == 1
    assert b"out_rest" in lib.ab_last_error(), lib.ab_last_error()
    assert lib.ab_tree_workspace_bytes(ctypes.byref(args)) == 0


@pytest.mark.parametrize("shape", [(3, 2, 8, 64), (2, 3, 2, 8, 64)])
def test_keys_and_values_in_one_place_are_not_moved(shape):
    """Each would move rows that the other one reads."""
    x, ints = torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="share no memory"):
        keep_drafts(PagedCache(x, x), ints[:2][None], ints[:1], ints[:2], ints, ints[:1])
