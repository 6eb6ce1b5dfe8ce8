"""Streaming operators on the GPU where tables, offsets and values are at the edge of what the interface allows."""
import pytest
import torch

from ab_attention.streaming import chunk_attention
from test_gpu_streaming import _cache, _check_chunk, _rand

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("page,window,sinks,frame,length", [(8, 10, 4, 1, 20), (16, 40, 4, 1, 60), (8, 20, 33, 1, 64), (8, 2, 1, 7, 28),
                                                            (8, 1000, 5, 1, 1025), (16, 1000, 5, 1, 1020)])
@pytest.mark.parametrize("new", [1, 3])
def test_chunk_holes_in_the_last_tile_of_sinks(page, window, sinks, frame, length, new):
    """A window that starts behind the sinks but in their last tile of 32 keys: every page of it that is missing is
    not seen, in short calls and in those whose keys are split (the last two)."""
    low = max(0, (length - new) // frame - window + 1) * frame
    assert sinks * frame < low < -(-sinks * frame // 32) * 32
    for hole in range(low // page, min(-(-sinks * frame // 32) * 32, length) // page):
        cache, table, lengths, offsets = _cache([new], [length], 2, 64, page, BF16)
        table[0, hole] = -1
        q = _rand((new, 4, 64), BF16, 3, 2.0)
        out, lse = chunk_attention(q, cache, table.cuda(), lengths.cuda(), offsets.cuda(), window=window, sinks=sinks, frame=frame,
                                   return_lse=True)
        _check_chunk(out, lse, q, cache, table, lengths, offsets, window, sinks, frame, BF16)
