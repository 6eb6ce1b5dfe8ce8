"""The streaming operators as they are used together: steps of a generation
against the whole sequence at once, captured graphs, other streams, several
threads."""
import threading

import pytest
import torch

from ab_attention.streaming import (PagedCache, StreamingAttention, append_cache, chunk_attention, rotary,
                                    window_attention)
from streaming_reference import HALF_STEP, attend, check_output, seen_mask

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _grid(frames, height, width, first=0):
    axes = torch.meshgrid(torch.arange(first, first + frames), torch.arange(height), torch.arange(width), indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], -1).cuda()


@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 1), (2, 0)])
@pytest.mark.parametrize("dtype,page", [(BF16, 64), (F16, 96)])
def test_generation_equals_the_whole_clip(window, sinks, dtype, page):
    """Two clips of frames of 6 x 16 tokens made a frame (or two, or none) a step, in two layers, on few pages: each
    token's output is that of window_attention over the rotated clip, but for the order of sums and splits."""
    frame, heads, kv, axes = 96, 6, 2, (44, 42, 42)
    plan = [(1, 1), (2, 0), (1, 1), (1, 1), (0, 2), (1, 1)]  # frames a step, of each clip
    frames = [sum(p[s] for p in plan) for s in range(2)]
    clips = [[_rand((frames[s] * frame, h, 128), dtype, 10 * s + i, 1.5) for i, h in enumerate((heads, kv, kv))] for s in range(2)]
    pages = 2 * -(-max(frames) * frame // page) if window is None else 2 * (-(-(window + 2 + sinks) * frame // page) + 2)
    stream = StreamingAttention(2, 2, kv, pages, page, window=window, sinks=sinks, frame=frame, axes=axes, dtype=dtype)
    got, done = [[[], []] for _ in range(2)], [0, 0]
    for step in plan:
        stream.begin([n * frame for n in step])
        rows = [slice(done[s] * frame, (done[s] + step[s]) * frame) for s in range(2)]
        packed = [torch.cat([clips[s][i][rows[s]] for s in range(2)]) for i in range(3)]
        positions = torch.cat([_grid(step[s], 6, 16, done[s]) for s in range(2)])
        for layer in range(2):
            q, k, v = packed if layer == 0 else (packed[0], packed[1], -packed[2])
            out = stream.attend(layer, q, k, v, positions)
            for s, part in enumerate(out.split([n * frame for n in step])):
                got[layer][s].append(part)
        done = [d + n for d, n in zip(done, step)]
    assert len(stream.free) + sum(len(h) for h in stream.held) == pages
    for s in range(2):
        q, k, v = (t.transpose(0, 1)[None] for t in clips[s])
        q, k = rotary(q, k, _grid(frames[s], 6, 16), axes)
        at = torch.arange(frames[s] * frame, device="cuda")
        o, _, spread = attend(q[0], k[0], v[0], seen_mask(at, at, window, sinks, frame))
        whole = window_attention(q, k, v, window=window, sinks=sinks, frame=frame)[0]
        for layer in range(2):
            out = torch.cat(got[layer][s]).transpose(0, 1)
            check_output(out, o if layer == 0 else -o, spread, dtype)
            # Two correct results: a rounding of P and one of the output apart on each side.
            room = 2 * HALF_STEP[dtype] * (spread + o.abs()) * 1.02 + 1e-4 * spread
            assert ((out.double() - (whole if layer == 0 else -whole).double()).abs() <= room).all()
    stream.finish(0)
    stream.finish(1)
    assert sorted(stream.free) == list(range(pages)) and stream.tokens == [0, 0]


def test_too_few_pages_change_nothing():
    stream = StreamingAttention(1, 2, 1, 4, 16, dim=64)
    stream.begin([30, 16])
    before = (list(stream.free), list(stream.tokens), [dict(h) for h in stream.held])
    with pytest.raises(ValueError, match="pages"):
        stream.begin([20, 17])
    assert before == (list(stream.free), list(stream.tokens), [dict(h) for h in stream.held])
    stream.finish(1)
    stream.begin([20, 0])
    with pytest.raises(ValueError, match="new tokens"):
        stream.begin([1])


def _decode_state(seed, lengths, page=32, heads=8, kv=2, dim=128):
    width = 16
    table = torch.randperm(len(lengths) * width, generator=torch.Generator().manual_seed(seed)).reshape(len(lengths), width)
    cache = PagedCache(*(_rand((len(lengths) * width, kv, page, dim), BF16, seed + i) for i in range(2)))
    n = len(lengths)
    return dict(cache=cache, table=table.to(torch.int32).cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                offsets=torch.arange(n + 1, dtype=torch.int32, device="cuda"), q=_rand((n, heads, dim), BF16, seed + 5),
                k=_rand((n, kv, dim), BF16, seed + 6), v=_rand((n, kv, dim), BF16, seed + 7),
                positions=torch.zeros((n, 1), dtype=torch.int32, device="cuda"))


def _decode(s):
    q, k = rotary(s["q"].transpose(0, 1)[None], s["k"].transpose(0, 1)[None], s["positions"], (128,), pairing="halves")
    q, k = q[0].transpose(0, 1), k[0].transpose(0, 1)
    append_cache(s["cache"], k, s["v"], s["table"], s["lengths"], s["offsets"])
    return chunk_attention(q, s["cache"], s["table"], s["lengths"], s["offsets"], window=200, sinks=3, return_lse=True)


def test_captured_decode_follows_its_inputs():
    """A captured step, replayed while sequences grow, against eager steps on a copy of the cache; two graphs of two
    states, replayed in turn."""
    states = [_decode_state(1, [1, 40, 300, 500]), _decode_state(2, [77, 400, 3, 129])]
    copies = [dict(s, cache=PagedCache(*(t.clone() for t in s["cache"]))) for s in states]
    graphs, outs = [], []
    for s in states:
        warm = dict(s, cache=PagedCache(*(t.clone() for t in s["cache"])))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _decode(warm)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_decode(s))
        graphs.append(graph)
    for step in range(5):
        for i, (s, copy) in enumerate(zip(states, copies)):
            for t in (s, copy):
                t["q"].copy_(_rand(t["q"].shape, BF16, 100 * step + i))
                t["k"].copy_(_rand(t["k"].shape, BF16, 200 * step + i))
                t["positions"].copy_((s["lengths"] - 1)[:, None])
            graphs[i].replay()
            want = _decode(copy)
            torch.cuda.synchronize()
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1]), step
            assert torch.equal(s["cache"].k, copy["cache"].k) and torch.equal(s["cache"].v, copy["cache"].v)
            s["lengths"].add_(1)
            if copy["lengths"] is not s["lengths"]:
                copy["lengths"].add_(1)


def _train(q, k, v, positions, do):
    a, b = rotary(q, k, positions, (32, 16, 16))
    out = window_attention(a, b, v, window=2, sinks=1, frame=48)
    return (out, *torch.autograd.grad(out, (q, k, v), do))


def test_captured_training_step():
    """Forward and backward in a graph, replayed with other values, against the eager step; run eagerly in between."""
    shape = (1, 4, 300, 64)
    leaves = [_rand((1, h, 300, 64), BF16, s).requires_grad_() for s, h in ((1, 4), (2, 2), (3, 2))]
    do, positions = _rand(shape, BF16, 4), torch.randint(0, 50, (300, 3), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _train(*leaves, positions, do)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _train(*leaves, positions, do)
    for step in range(4):
        with torch.no_grad():
            for i, t in enumerate((*leaves, do)):
                t.copy_(_rand(t.shape, BF16, 50 * step + i))
        graph.replay()
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        want = _train(*fresh, positions, do)
        torch.cuda.synchronize()
        for got, w in zip(captured, want):
            assert torch.equal(got, w), step


def test_streams_and_threads():
    """Calls on streams of their own, from threads of their own, give the bits of one call after the other."""
    states = [_decode_state(10 + i, [5 + i, 300 - i, 511]) for i in range(4)]
    want = [_decode(dict(s, cache=PagedCache(*(t.clone() for t in s["cache"])))) for s in states]
    leaves = [[_rand((1, 4, 260, 64), F16, 5 * i + j).requires_grad_() for j in range(3)] for i in range(4)]
    grads = [torch.autograd.grad(window_attention(*t, window=70, sinks=2).sum(), t) for t in leaves]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    out = _decode(states[i])
                    g = torch.autograd.grad(window_attention(*leaves[i], window=70, sinks=2).sum(), leaves[i])
            stream.synchronize()
            got[i] = (out, g)
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for (out, g), w, wg in zip(got, want, grads):
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
        assert all(torch.equal(a, b) for a, b in zip(g, wg))


def test_split_and_whole_rows_agree():
    """A token over a long cache is split over workgroups; beside 600 other sequences it is not: the same attention."""
    lengths = [8000] + [33] * 600
    width = -(-8000 // 64)
    table = torch.full((601, width), -1, dtype=torch.int32)
    table[0] = torch.arange(width, dtype=torch.int32)
    table[1:, 0] = torch.arange(width, width + 600, dtype=torch.int32)
    cache = PagedCache(*(_rand((width + 600, 1, 64, 128), BF16, s) for s in (1, 2)))
    q = _rand((601, 4, 128), BF16, 3, 2.0)
    dev = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    whole = chunk_attention(q, cache, table.cuda(), dev(*lengths), dev(*range(602)), return_lse=True)
    split = chunk_attention(q[:1], cache, table[:1].cuda(), dev(8000), dev(0, 1), return_lse=True)
    at = torch.arange(8000, device="cuda")
    k, v = (t[at // 64, :, at % 64].transpose(0, 1) for t in cache)
    o, lse, spread = attend(q[0][:, None], k, v, torch.ones((1, 8000), dtype=torch.bool, device="cuda"))
    for out, got in (whole, split):
        check_output(out[0][:, None], o, spread, BF16)
        assert (got[0].double() - lse[:, 0]).abs().max() <= 1e-4
