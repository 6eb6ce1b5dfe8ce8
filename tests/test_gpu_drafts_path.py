"""The operators of drafted tokens as they are used together: whole steps, forks, graphs, streams."""
import random

import pytest
import torch

from ab_attention.streaming import (PagedCache, StreamingAttention, append_cache, draft_tree, keep_drafts, rotary, tree_attention,
                                    verify_drafts)
from drafts_reference import make_tree
from streaming_reference import attend, check_output, seen_mask

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


class _Model:
    """Layers whose Q, K and V are rows of tables by token: what a token's output has to be follows from the tokens before it."""

    def __init__(self, layers, heads, kv, vocab, dtype, window, sinks):
        self.q = _rand((layers, vocab, heads, 64), dtype, 1, 1.5)
        self.k, self.v = (_rand((layers, vocab, kv, 64), dtype, s) for s in (2, 3))
        self.layers, self.vocab, self.how, self.dtype = layers, vocab, (window, sinks, 1), dtype

    def step(self, stream, tokens, positions):
        tokens = torch.tensor(tokens, device="cuda")
        return [stream.attend(i, self.q[i, tokens], self.k[i, tokens], self.v[i, tokens], positions[:, None]) for i in range(self.layers)]

    def check(self, tokens, outputs):
        """outputs[layer][i]: of the i-th token."""
        n = len(tokens)
        at, tokens = torch.arange(n, device="cuda"), torch.tensor(tokens, device="cuda")
        for i in range(self.layers):
            q, k = rotary(self.q[i, tokens].transpose(0, 1)[None], self.k[i, tokens].transpose(0, 1)[None], at[:, None], (64,))
            o, _, spread = attend(q[0], k[0], self.v[i, tokens].transpose(0, 1), seen_mask(at, at, *self.how))
            check_output(torch.stack(outputs[i]).transpose(0, 1), o, spread, self.dtype)


@pytest.mark.parametrize("window,sinks,page,dtype,drawn", [(None, 0, 8, BF16, True), (23, 3, 16, F16, False), (5, 0, 8, BF16, True)])
def test_text_made_by_drafts(window, sinks, page, dtype, drawn):
    """Three sequences in steps of drafts, one of them pausing now and then: every kept token's output is that of plain
    attention over the tokens that were kept."""
    vocab, sequences = 11, 3
    model = _Model(2, 4, 2, vocab, dtype, window, sinks)
    stream = StreamingAttention(2, sequences, 2, 60, page, dim=64, window=window, sinks=sinks, axes=(64,), dtype=dtype)
    rng = random.Random(5)
    gen = torch.Generator("cuda").manual_seed(6)
    last, text = [1, 2, 3], [[] for _ in range(sequences)]
    outputs = [[[] for _ in range(2)] for _ in range(sequences)]
    taken = 0
    for step in range(25):
        new = [0 if rng.random() < 0.15 else rng.randint(1, 14) for _ in range(sequences)]
        trees = [make_tree(n, rng.choice([0, 1, 2, 3]), step) for n in new]
        rows = sum(new)
        taken += sum(n > 0 for n in new)
        if rows == 0:
            continue
        target, draft = (torch.rand((rows, vocab), generator=gen, device="cuda").pow(2) for _ in range(2))
        target, draft = target / target.sum(-1, keepdim=True), draft / draft.sum(-1, keepdim=True)
        draft = 0.3 * draft + 0.7 * target
        tokens, at = [], 0
        for s, tree in enumerate(trees):
            tokens += [last[s] if j == 0 else int(draft[at + p].multinomial(1, generator=gen)) for j, p in enumerate(tree)]
            at += len(tree)
        stream.begin(new, trees)
        out = model.step(stream, tokens, stream.tree.positions)
        kept = verify_drafts(target, draft if drawn else None, torch.tensor(tokens, device="cuda"),
                             torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda"), stream.offsets,
                             torch.rand(rows, generator=gen, device="cuda"))
        counts = stream.keep(kept.path, kept.counts)
        path, at = kept.path.tolist(), 0
        for s, (n, count) in enumerate(zip(new, counts)):
            for j in path[at:at + count]:
                text[s].append(tokens[at + j])
                for layer in range(2):
                    outputs[s][layer].append(out[layer][at + j])
            if n:
                last[s] = int(kept.next[s])
            at += n
        assert stream.tokens == [len(t) for t in text]
        held = [page for h in stream.held for page in h.values()]
        assert sorted(held + stream.free) == list(range(60))
    assert sum(len(t) for t in text) > taken  # some drafts were kept
    for s in range(sequences):
        model.check(text[s], outputs[s])


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
def test_forks_go_their_own_ways(window, sinks):
    """One beginning continued in three ways, two of them in the same step: shared pages are copied by those who write
    first, and given back once nobody has them."""
    model = _Model(2, 2, 1, 9, BF16, window, sinks)
    stream = StreamingAttention(2, 3, 1, 24, 8, dim=64, window=window, sinks=sinks, axes=(64,))
    rng = random.Random(1)
    text, outputs = [[] for _ in range(3)], [[[], []] for _ in range(3)]

    def step(new):
        tokens = [[rng.randrange(9) for _ in range(n)] for n in new]
        first = list(stream.tokens)
        stream.begin(new)
        positions = torch.tensor([first[s] + i for s, n in enumerate(new) for i in range(n)], device="cuda")
        out = model.step(stream, sum(tokens, []), positions)
        at = 0
        for s, n in enumerate(new):
            text[s] += tokens[s]
            for layer in range(2):
                outputs[s][layer] += out[layer][at:at + n]
            at += n
        owned = [0] * 24
        for held in stream.held:
            for page in held.values():
                owned[page] += 1
        assert owned == stream.owners and sorted(stream.free) == [p for p in range(24) if not owned[p]]

    step([13, 0, 0])
    for into in (1, 2):
        stream.fork(0, into)
        text[into], outputs[into] = list(text[0]), [list(o) for o in outputs[0]]
    assert len(stream.free) == 24 - 2
    with pytest.raises(ValueError, match="after begin"):
        stream.attend(0, *[_rand((1, 1, 64), BF16, 1)] * 3)
    step([2, 1, 0])    # two write into the shared page: both get copies, the third has it alone
    step([0, 0, 5])
    step([9, 3, 1])
    stream.finish(1)
    text[1], outputs[1] = [], [[], []]
    stream.fork(2, 1)
    text[1], outputs[1] = list(text[2]), [list(o) for o in outputs[2]]
    for _ in range(6):
        step([rng.randint(0, 6) for _ in range(3)])
    for s in range(3):
        model.check(text[s], outputs[s])
    for s in range(3):
        stream.finish(s)
    assert sorted(stream.free) == list(range(24)) and not any(stream.owners)


def test_too_few_pages_for_copies_change_nothing():
    stream = StreamingAttention(1, 2, 1, 3, 8, dim=64)
    stream.begin([20, 0])
    stream.fork(0, 1)
    before = (list(stream.free), list(stream.tokens), [dict(h) for h in stream.held], list(stream.owners))
    with pytest.raises(ValueError, match="1 more pages are needed, 0 are free"):
        stream.begin([1, 1])
    assert before == (stream.free, stream.tokens, stream.held, stream.owners)
    stream.finish(1)
    stream.begin([4, 0])


def _state(seed, batch=3, n=9, vocab=1500):
    rng = random.Random(seed)
    page, width = 8, 12
    trees = [make_tree(n, 2, seed + b) for b in range(batch)]
    table = torch.randperm(batch * width, generator=torch.Generator().manual_seed(seed)).reshape(batch, width).to(torch.int32)
    s = dict(k_cache=_rand((2, batch * width, 2, page, 64), BF16, seed), v_cache=_rand((2, batch * width, 2, page, 64), BF16, seed + 1),
             table=table.cuda(), offsets=torch.arange(0, batch * n + 1, n, dtype=torch.int32, device="cuda"),
             parents=torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda"),
             lengths=torch.tensor([n + rng.randint(0, 40) for _ in range(batch)], dtype=torch.int32, device="cuda"),
             tokens=torch.zeros(batch * n, dtype=torch.int64, device="cuda"))
    _refill(s, seed)
    s["target"], s["draft"] = (torch.rand((batch * n, vocab), device="cuda").softmax(-1) for _ in range(2))
    _refill(s, seed)
    return s


def _refill(s, seed):
    """New values in the same tensors."""
    rows = s["tokens"].shape[0]
    gen = torch.Generator("cuda").manual_seed(seed)
    for i, (name, heads) in enumerate((("q", 4), ("k", 2), ("v", 2))):
        x = _rand((2, rows, heads, 64), BF16, seed * 7 + i)
        s[name] = s[name].copy_(x) if name in s else x
    u = torch.rand(rows, generator=gen, device="cuda")
    s["uniforms"] = s["uniforms"].copy_(u) if "uniforms" in s else u
    if "target" in s:
        s["target"].copy_(torch.randn(s["target"].shape, generator=gen, device="cuda").mul(3).softmax(-1))
        s["draft"].copy_((s["target"].log() + torch.randn(s["target"].shape, generator=gen, device="cuda")).softmax(-1))
        s["tokens"].copy_(s["draft"][(torch.arange(rows, device="cuda") // 9 * 9 + s["parents"].clamp_min(0))].multinomial(1, generator=gen)[:, 0])


def _step(s):
    where = s["table"], s["lengths"], s["offsets"]
    tree, out = draft_tree(s["parents"], s["lengths"], s["offsets"]), []
    for layer in range(2):
        cache = PagedCache(s["k_cache"][layer], s["v_cache"][layer])
        append_cache(cache, s["k"][layer], s["v"][layer], *where)
        out += tree_attention(s["q"][layer], cache, *where, tree, window=30, sinks=2, return_lse=True)
    kept = verify_drafts(s["target"], s["draft"], s["tokens"], s["parents"], s["offsets"], s["uniforms"])
    keep_drafts(PagedCache(s["k_cache"], s["v_cache"]), *where, kept.path, kept.counts)
    return [*tree, *out, *kept]


def _copy(s):
    return {name: t.clone() for name, t in s.items()}


def test_captured_steps_follow_their_inputs():
    """Two captured steps of two states, replayed in turn while their inputs change, against eager steps on copies, whose
    values are used between the replays."""
    states = [_state(1), _state(2)]
    copies = [_copy(s) for s in states]
    graphs, outs = [], []
    for s in states:
        warm = _copy(s)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(warm)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(s))
        graphs.append(graph)
    for step in range(5):
        for i, (s, copy) in enumerate(zip(states, copies)):
            for t in (s, copy):
                _refill(t, 10 * step + i)
            graphs[i].replay()
            want = _step(copy)
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), step
            assert torch.equal(s["k_cache"], copy["k_cache"]) and torch.equal(s["v_cache"], copy["v_cache"])
            for t in (s, copy):  # the sequences go on behind what was kept
                t["lengths"].add_(want[-2]).sub_(9).clamp_(max=60).add_(9)


def test_two_streams_at_once():
    """Steps of two states on streams of their own, one behind the other on each, against the same on one stream."""
    states = [_state(3, n=9), _state(4, n=9)]
    copies = [_copy(s) for s in states]
    want = [[_step(s) for _ in range(4)] for s in copies]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for i, s in enumerate(states):
            with torch.cuda.stream(streams[i]):
                got[i].append(_step(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert all(torch.equal(t, u) for t, u in zip(x, y))
    assert all(torch.equal(s["k_cache"], c["k_cache"]) for s, c in zip(states, copies))
