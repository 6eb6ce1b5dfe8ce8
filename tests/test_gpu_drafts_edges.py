"""Drafted tokens on the GPU: calls at the edge of what is allowed."""
import math

import pytest
import torch

from ab_attention.streaming import PagedCache, draft_tree, tree_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,new", [(64, 1, 3), (128, 4, 66)])
def test_more_tiles_of_keys_than_float32_counts(dim, heads, new):
    """A sequence of 17,026,881 tiles of keys, beside one that brings nothing: rounded to float32 their 64th part is a
    step short, so that 64 such parts would leave one over. All keys are 0 and all values alike, so every row's output
    is the value itself (its sum and that of the weights round alike), and its normaliser the number of keys it sees."""
    length, page = 17026881 * 32, 8192
    cache = PagedCache(torch.zeros((1, 1, page, dim), dtype=torch.bfloat16, device="cuda"),
                       torch.empty((1, 1, page, dim), dtype=torch.bfloat16, device="cuda"))
    value = torch.tensor([1.0, -0.5, 2.0, -4.0], device="cuda").repeat(dim // 4).bfloat16()
    cache.v[:] = value
    table = torch.zeros((2, -(-length // page)), dtype=torch.int32, device="cuda")
    lengths, offsets = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([length, 5], [0, new, new]))
    tree = draft_tree(torch.arange(-1, new - 1, dtype=torch.int32, device="cuda"), lengths, offsets)
    q = torch.ones((new, heads, dim), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 7.0)
    o, lse = tree_attention(q, cache, table, lengths, offsets, tree, return_lse=True, out=out)
    assert torch.equal(o, value.expand_as(o))
    # Up to 65 parts' sums, added in float32, are off by half a step each; the logarithm, near 29, by two steps of
    # 2^-19, and its sum with the reference by half of one.
    seen = torch.arange(length - new + 1, length + 1, dtype=torch.float64, device="cuda")
    bound = 65 * 2 ** -24 / math.log(2) + 2.5 * 2 ** -19
    assert ((lse.double() - seen.log2()[:, None]).abs() < bound).all()
