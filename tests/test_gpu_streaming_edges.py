"""Streaming operators on the GPU where tables, offsets and values are at the edge of what the interface allows."""
import math

import pytest
import torch

from ab_attention.streaming import PagedCache, StreamingAttention, append_cache, chunk_attention, window_attention
from streaming_reference import attend, check_output, seen_mask
from test_gpu_streaming import _cache, _check_chunk, _rand

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


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


def _under_a_sink(n, heads, drop, spread, seed=0):
    """q, k, v [1, heads, n, 64] in fp16 of a first key that is `drop` (base 2) above the others and has no value."""
    q, k, v = (_rand((1, heads, n, 64), F16, seed + s) for s in (1, 2, 3))
    k *= spread
    q[..., 0], k[..., 0] = 4, 0
    k[:, :, 0] = 0
    k[:, :, 0, 0] = drop * 8 / (4 * math.log2(math.e))
    v[:, :, 0] = 0
    return q, k, v


@pytest.mark.parametrize("drop,spread", [(12, 1.0), (18, 0.0), (18, 1.0), (21.6, 0.0), (21.6, 1.0), (24, 0.0), (24, 1.0)])
def test_fp16_output_of_small_probabilities(drop, spread):
    """A sink that takes nearly all the weight and gives nothing: the output is the sum of thousands of weights that are
    each rounded relative to their own size. Whole and split rows, tensors and caches."""
    for n, heads in ((4000, 17), (1300, 1)):
        q, k, v = _under_a_sink(n, heads, drop, spread)
        at = torch.arange(n, device="cuda")
        o, _, size = attend(q[0], k[0], v[0], seen_mask(at, at, None, 0, 1))
        check_output(window_attention(q, k, v)[0], o, size, F16)
        check_output(window_attention(q.clone().requires_grad_(), k, v)[0].detach(), o, size, F16)
    width = 4000 // 16
    cache = PagedCache(*(t[0, :1].reshape(1, width, 16, 64).transpose(0, 1).contiguous() for t in _under_a_sink(4000, 1, drop, spread)[1:]))
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(width, dtype=torch.int32, device="cuda")[None]
    for new, group in ((1, 8), (3000, 16)):
        q = _rand((new, group, 64), F16, 9)
        q[..., 0] = 4
        out, lse = chunk_attention(q, cache, table, dev(4000), dev(0, new), return_lse=True)
        _check_chunk(out, lse, q, cache, table.cpu(), dev(4000), dev(0, new), None, 0, 1, F16)


def test_append_and_chunk_agree_on_offsets_beyond_the_rows():
    """Offsets past the packed rows count as their end, those below 0 as 0: append_cache and chunk_attention place the
    rows alike, and write nothing else."""
    cache, table, lengths, offsets = _cache([3, 4], [50, 70], 2, 64, 16, BF16)
    k, v, q = (_rand((7, h, 64), BF16, s, 2.0) for s, h in ((1, 2), (2, 2), (3, 4)))
    dev = [table.cuda(), lengths.cuda()]
    want = append_cache(PagedCache(*(t.clone() for t in cache)), k, v, *dev, offsets.cuda())
    o, lse = chunk_attention(q, want, *dev, offsets.cuda(), return_lse=True)
    for first, last in ((0, 9), (0, 2 ** 31 - 1), (-2, 7), (-2 ** 31, 40)):
        far = torch.tensor([first, 3, last], dtype=torch.int32, device="cuda")
        got = append_cache(PagedCache(*(t.clone() for t in cache)), k, v, *dev, far)
        assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v), (first, last)
        guard = torch.full((20, 4, 64), 3.0, dtype=BF16, device="cuda")
        out, l = chunk_attention(q, got, *dev, far, return_lse=True, out=guard[6:13])
        assert torch.equal(out, o) and torch.equal(l, lse), (first, last)
        assert (guard[:6] == 3).all() and (guard[13:] == 3).all()
    _check_chunk(o, lse, q, want, table, lengths, offsets, None, 0, 1, BF16)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_chunk_values_that_are_not_finite_whatever_the_split(value):
    """A key whose weight is far below float32's smallest, with a value that is not finite: the query sees it, alone in
    the call (its keys split over workgroups) and beside 600 others (not split)."""
    n, width = 8000, 125
    table = torch.full((601, width), -1, dtype=torch.int32)
    table[0] = torch.arange(width, dtype=torch.int32)
    table[1:, 0] = torch.arange(width, width + 600, dtype=torch.int32)
    cache = PagedCache(*(_rand((width + 600, 1, 64, 128), BF16, s) for s in (1, 2)))
    q = _rand((601, 1, 128), BF16, 3)
    q[0, 0, 0], cache.k[..., 0] = 16, 0
    cache.k[100, 0, 7, 0] = 160  # position 6407: 16 * 160 / sqrt(128) * log2(e), some 326 above the others
    cache.v[3, 0, 9, 5] = value  # position 201
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    whole = chunk_attention(q, cache, table.cuda(), dev(n, *[33] * 600), dev(*range(602)))
    split = chunk_attention(q[:1], cache, table[:1].cuda(), dev(n), dev(0, 1))
    for out in (whole, split):
        assert not out[0, 0, 5].isfinite()
        rest = [i for i in range(128) if i != 5]
        assert torch.equal(out[0, 0, rest], cache.v[100, 0, 7, rest])


def test_saved_tensors_that_are_written_again_are_refused():
    """Keys that a gradient still needs, then written as a cache by append_cache or as chunk_attention's out."""
    cache, *where = _cache([4], [10], 2, 64, 16, BF16)
    where = [t.cuda() for t in where]
    where[0].zero_()
    x = _rand((4, 2, 64), BF16, 1)

    def used():
        q, kept = _rand((1, 2, 16, 64), BF16, 3).requires_grad_(), _rand((1, 2, 16, 64), BF16, 2)
        return window_attention(q, kept, kept), kept

    out, kept = used()
    append_cache(PagedCache(kept, kept.clone()), x, x, *where)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out, kept = used()
    chunk_attention(x, cache, *where, out=kept[0, :, :4].transpose(0, 1))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("new,total", [([1, 1], [6000, 130]), ([1, 900, 77], [300, 1100, 4000])])
def test_chunk_out_over_its_queries(new, total):
    """out may be q itself: whole rows and split ones."""
    cache, *where = _cache(new, total, 2, 64, 16, BF16)
    where = [t.cuda() for t in where]
    q = _rand((sum(new), 8, 64), BF16, 3, 2.0)
    want = chunk_attention(q, cache, *where, window=3000, sinks=4)
    assert chunk_attention(q, cache, *where, window=3000, sinks=4, out=q) is q
    assert torch.equal(q, want)


def test_streaming_steps_are_not_captured():
    """A captured attend would go on reading the page table of the step that it was captured in."""
    stream = StreamingAttention(1, 1, 2, 4, 16, dim=64)
    stream.begin([5])
    x = _rand((5, 2, 64), BF16, 1)
    want = stream.attend(0, x, x, x)
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(3, device="cuda")
    with torch.cuda.graph(graph):
        for call in (lambda: stream.begin([5]), lambda: stream.attend(0, x, x, x)):
            with pytest.raises(ValueError, match="captured"):
                call()
        y.add_(1)
    graph.replay()
    assert (y == 1).all() and torch.equal(stream.attend(0, x, x, x), want)
