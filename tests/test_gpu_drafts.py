"""The operators of drafted tokens on the GPU against their plain forms in 64 bits."""
import math
import random

import pytest
import torch

from ab_attention.streaming import (DraftTree, PagedCache, append_cache, chunk_attention, copy_pages, draft_tree,
                                    keep_drafts, tree_attention, verify_drafts)
from drafts_reference import make_tree, tree_attend, tree_tensors, verify
from streaming_reference import check_lse, check_output, logit_size

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(new, first=0):
    offsets = [first]
    for n in new:
        offsets.append(offsets[-1] + n)
    return _ints(offsets)


def _packed(trees, before=0, behind=0):
    return _ints([77] * before + [p for tree in trees for p in tree] + [77] * behind)


# ---- the tree -----------------------------------------------------------------


@pytest.mark.parametrize("branch", [-1, 0, 1, 2, 3])
@pytest.mark.parametrize("sizes", [(1,), (2, 0, 3), (63, 64, 65), (26,) * 70, (300, 1, 129), (1025,), (5, 4500)])
def test_draft_tree(sizes, branch):
    trees = [make_tree(n, branch, s) for s, n in enumerate(sizes)]
    lengths = [n + 7 * s - 3 for s, n in enumerate(sizes)]  # the first sequence lacks three tokens
    before, behind = 3, 70
    tree = draft_tree(_packed(trees, before, behind), _ints(lengths), _offsets(sizes, before))
    at = before
    assert not tree.positions[:before].any() and not tree.near[:before].any() and (tree.above[:before] == -1).all()
    for its, length in zip(trees, lengths):
        positions, near, above = tree_tensors(its, length - len(its))
        rows = slice(at, at + len(its))
        assert tree.positions[rows].tolist() == positions
        assert [x & 2 ** 64 - 1 for x in tree.near[rows].tolist()] == near
        assert tree.above[rows].tolist() == above
        at += len(its)
    assert not tree.positions[at:].any() and not tree.near[at:].any() and (tree.above[at:] == -1).all()


def test_draft_tree_of_nothing():
    tree = draft_tree(_ints([]), _ints([5]), _ints([0, 0]))
    assert [t.shape[0] for t in tree] == [0, 0, 0]
    tree = draft_tree(_ints([0, 1]), _ints([]), _ints([0]))
    assert tree.positions.tolist() == [0, 0] and tree.above.tolist() == [-1, -1]


# ---- attention ----------------------------------------------------------------


class _Call:
    """Caches and a page table of sequences with `new` tokens behind `cached` ones."""

    def __init__(self, new, cached, heads, kv_heads, dim, page, dtype, seed, branch=2, token_major=False, before=0, behind=0):
        self.new, self.lengths_ = new, [n + c for n, c in zip(new, cached)]
        needed = [-(-length // page) for length in self.lengths_]
        pages = sum(needed) + 2
        shape = (pages, page, kv_heads, dim) if token_major else (pages, kv_heads, page, dim)
        k, v = (_rand(shape, dtype, seed + i) for i in range(2))
        self.cache = PagedCache(*(t.transpose(1, 2) if token_major else t for t in (k, v)))
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        self.rows_ = []
        for count in needed:
            self.rows_.append([order.pop() for _ in range(count)])
        width = max(1, max(needed))
        self.table = _ints([row + [-1] * (width - len(row)) for row in self.rows_])
        self.lengths, self.offsets = _ints(self.lengths_), _offsets(new, before)
        self.q = _rand((before + sum(new) + behind, heads, dim), dtype, seed + 2, 2.0)
        self.trees = [make_tree(n, branch, seed + s) for s, n in enumerate(new)]
        self.parents = _packed(self.trees, before, behind)
        self.before = before

    def tree(self):
        return draft_tree(self.parents, self.lengths, self.offsets)

    def run(self, **kw):
        return tree_attention(self.q, self.cache, self.table, self.lengths, self.offsets, self.tree(), return_lse=True, **kw)

    def check(self, o, lse, **kw):
        dtype, at = self.q.dtype, self.before
        size = logit_size(self.q, self.cache.k, kw.get("scale"))
        for n, length, row, tree in zip(self.new, self.lengths_, self.table, self.trees):
            if n == 0:
                continue
            rows = slice(at, at + n)
            ref_o, ref_lse, spread = tree_attend(self.q[rows], self.cache, row, length, tree, **kw)
            check_output(o[rows], ref_o, spread, dtype)
            check_lse(lse[rows], ref_lse, self.q.shape[-1], size)
            at += n


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 3, 3), (128, 1, 1), (64, 16, 1)])
@pytest.mark.parametrize("new,cached,page,branch", [
    ((1,), (0,), 8, 1), ((5,), (0,), 16, 2), ((26,), (101,), 16, 3), ((64, 1, 33), (0, 250, 63), 64, -1),
    ((65, 0, 130), (31, 5, 2), 32, 0), ((300,), (77,), 8, -1), ((17,) * 67, tuple(range(67)), 24, 2),
    ((1, 2, 0) * 110, (3, 700, 9) * 110, 32, 1)])
def test_tree_attention(dtype, dim, heads, kv_heads, new, cached, page, branch):
    call = _Call(new, cached, heads, kv_heads, dim, page, dtype, 11, branch)
    o, lse = call.run()
    call.check(o, lse)


@pytest.mark.parametrize("window,sinks,frame", [(1, 0, 1), (4, 0, 1), (3, 2, 1), (40, 4, 1), (40, 130, 1), (2, 1, 10), (1, 0, 48),
                                                (5, 1, 7), (10 ** 12, 10 ** 12, 1), (200, 300, 1)])
@pytest.mark.parametrize("new,cached,branch", [((26, 9), (150, 3), 2), ((90,), (20,), 1), ((40, 70), (0, 333), -1), ((130,), (65,), 0)])
def test_tree_attention_windows(window, sinks, frame, new, cached, branch):
    """Windows that end among the cached tokens, among the drafts, before both."""
    call = _Call(new, cached, 4, 2, 64, 16, BF16, 5, branch, token_major=True)
    how = dict(window=window, sinks=sinks, frame=frame)
    o, lse = call.run(**how)
    call.check(o, lse, **how)


@pytest.mark.parametrize("window,sinks,frame", [(None, 0, 1), (4, 0, 1), (40, 130, 1), (5, 1, 7)])
@pytest.mark.parametrize("heads,new,cached,branch", [(8, (26, 80), (1500, 3), 2), (8, (17,), (41,), 0), (5, (33, 0, 128), (70, 5, 0), -1),
                                                     (1, (2200,), (21,), 3)])
def test_tree_attention_many_rows(heads, new, cached, branch, window, sinks, frame):
    """Sequences of more than 128 rows: token and query head of the group."""
    call = _Call(new, cached, heads, 1, 128, 16, BF16, 17, branch)
    how = dict(window=window, sinks=sinks, frame=frame)
    call.check(*call.run(**how), **how)
    call.table[0, 1] = -1
    call.table[0, (cached[0] + new[0] // 2) // 16] = 10 ** 9  # a page of drafts
    call.check(*call.run(**how), **how)


@pytest.mark.parametrize("cached", [3000, 9001])
@pytest.mark.parametrize("n,branch", [(1, 1), (40, 3), (200, 0)])
def test_tree_attention_split(cached, n, branch):
    """Few rows over many keys: parts of the keys are added up."""
    call = _Call((n,), (cached,), 4, 1, 128, 64, BF16, 21, branch)
    o, lse = call.run()
    call.check(o, lse)
    call.check(*call.run(window=2500, sinks=5), window=2500, sinks=5)


@pytest.mark.parametrize("new,cached", [((3, 0, 7, 1) * 25, (9000, 5, 40, 2500) * 25), ((0,) * 70 + (40,) + (0,) * 60, (1,) * 70 + (20000,) + (3,) * 60),
                                        ((40, 33) * 40, (700, 9) * 40), ((90, 1, 0) * 50, (5000, 3, 1) * 50),
                                        ((1, 0, 2) * 500, (0, 9, 30) * 500), ((2, 0, 0, 1) * 1050 + (0,), (5, 1, 2, 0) * 1050 + (4,))])
def test_tree_attention_many_sequences(new, cached):
    """Sequences that share one K/V head, more than a wave, a workgroup and 64 waves have lanes; a few of them long."""
    call = _Call(new, cached, 4, 1, 128, 64, BF16, 23, 2, before=2, behind=1)
    out = torch.full_like(call.q, 7.0)
    o, lse = call.run(out=out)
    assert (o[:2] == 7).all() and (o[-1:] == 7).all()
    call.check(o, lse)


@pytest.mark.parametrize("heads,kv_heads,n,branch", [(1, 1, 1100, 0), (2, 2, 1500, -1), (8, 1, 4300, 1), (3, 1, 3100, 0)])
@pytest.mark.parametrize("cached", [0, 21, 70])
def test_tree_attention_long_drafts(heads, kv_heads, n, branch, cached):
    """More drafts than a workgroup keeps the lines of."""
    call = _Call((n,), (cached,), heads, kv_heads, 64, 64, BF16, 13, branch)
    call.check(*call.run())
    call.check(*call.run(window=40, sinks=3), window=40, sinks=3)


@pytest.mark.parametrize("dim,new,cached", [(128, (70, 5), (40, 900)), (64, (1,), (5000,)), (64, (200,), (31,))])
def test_a_chain_is_a_chunk(dim, new, cached):
    call = _Call(new, cached, 6, 2, dim, 16, BF16, 3, 1)
    # Both cut the keys in parts and tiles of their own, so the same sums are made in another order: each is within the
    # bound of one call.
    for how in ({}, dict(window=50, sinks=4), dict(window=3)):
        o, lse = call.run(**how)
        o2, lse2 = chunk_attention(call.q, call.cache, call.table, call.lengths, call.offsets, return_lse=True, **how)
        call.check(o, lse, **how)
        call.check(o2, lse2, **how)


@pytest.mark.parametrize("pages,width", [(0, 4), (3, 0), (0, 0)])
@pytest.mark.parametrize("batch", [2, 70])
def test_a_cache_without_keys(pages, width, batch):
    cache = PagedCache(*(torch.zeros((pages, 2, 16, 128), dtype=BF16, device="cuda") for _ in range(2)))
    new = (3, 50) * (batch // 2)
    lengths, offsets = _ints([20] * batch), _offsets(new)
    tree = draft_tree(_packed([make_tree(n, 2, 1) for n in new]), lengths, offsets)
    q = _rand((sum(new), 4, 128), BF16, 1)
    o, lse = tree_attention(q, cache, torch.zeros((batch, width), dtype=torch.int32, device="cuda"), lengths, offsets, tree, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    kept = keep_drafts(cache, torch.zeros((batch, width), dtype=torch.int32, device="cuda"), lengths, offsets,
                       torch.full_like(tree.above, 1), _ints([2] * batch))
    assert kept is cache and not any(t.any() for t in cache)


def test_rows_of_no_sequence_stay():
    call = _Call((9, 0, 20), (30, 4, 0), 4, 2, 64, 8, F16, 8, 2, before=3, behind=5)
    out = torch.full_like(call.q, 7.0)
    o, lse = call.run(out=out)
    assert o is out and (out[:3] == 7).all() and (out[-5:] == 7).all()
    call.check(o, lse)


def test_missing_pages_and_strides():
    call = _Call((12, 30), (100, 60), 4, 2, 64, 8, BF16, 9, 3)
    call.table[0, 2] = -1
    call.table[0, 13] = 10 ** 9   # a page of drafts
    call.table[1, 0] = -5
    o, lse = call.run()
    call.check(o, lse)
    # Q and out as slices of wider rows, heads and tokens in the other order.
    wide = _rand((4, 42, 3 * 64), BF16, 2)
    call.q = wide[..., 64:128].transpose(0, 1)
    out = torch.zeros((42, 4, 64 * 2), dtype=BF16, device="cuda")[..., 64:]
    o, lse = call.run(out=out)
    assert o is out
    call.check(o, lse)


@pytest.mark.parametrize("heads", [4, 14])
def test_drafts_that_are_not_seen_may_hold_anything(heads):
    """Infinities and NaN in another line's keys and values reach no token that does not follow them."""
    call = _Call((40,), (21,), heads, 2, 128, 16, BF16, 4, 2)
    ref_o, ref_lse, spread = tree_attend(call.q, call.cache, call.table[0], 61, call.trees[0])
    size = logit_size(call.q, call.cache.k)
    bad = 17
    at = 21 + bad
    entry = call.rows_[0][at // 16]
    keep = [t[entry, :, at % 16].clone() for t in call.cache]
    touched = [i for i in range(40) if bad in _line(call.trees[0], i)]
    for k_value, v_value in ((math.inf, math.nan), (math.nan, -math.inf), (3.0, math.inf)):
        call.cache.k[entry, :, at % 16] = k_value
        call.cache.v[entry, :, at % 16] = v_value
        o, lse = call.run()
        others = [i for i in range(40) if i not in touched]
        check_output(o[others], ref_o[others], spread[others], BF16)
        check_lse(lse[others], ref_lse[others], 128, size)
        assert not torch.isfinite(o[touched]).any()
        for t, kept in zip(call.cache, keep):
            t[entry, :, at % 16] = kept
    # Behind the last token of the sequence.
    clean = call.run()
    at = 61
    entry = call.rows_[0][at // 16]
    call.cache.k[entry, :, at % 16:] = math.nan
    call.cache.v[entry, :, at % 16:] = math.nan
    assert torch.equal(call.run()[0], clean[0])


def _line(tree, i):
    line = []
    while i >= 0:
        line.append(i)
        i = tree[i] if tree[i] < i else -1
    return line


def test_lengths_below_the_new_tokens():
    """Tokens that would lie before the cache's first place are not there."""
    call = _Call((10, 80), (0, 0), 2, 1, 64, 8, BF16, 6, 2)
    call.lengths_ = [4, 70]
    call.lengths = _ints(call.lengths_)
    o, lse = call.run()
    call.check(o, lse)
    call.lengths_ = [0, 70]
    call.lengths = _ints(call.lengths_)
    o, lse = call.run()
    assert not o[:10].any() and torch.isinf(lse[:10]).all()


def test_a_tree_of_other_values_stays_inside():
    """Whatever the tree holds, nothing outside of the call's memory is reached, and the call ends."""
    call = _Call((70, 30), (20, 40), 4, 2, 64, 16, BF16, 7, 2)
    gen = torch.Generator("cuda").manual_seed(1)
    for low, high in ((-2 ** 31, 2 ** 31 - 1), (-1, 200)):
        positions, above = (torch.randint(low, high, (100,), generator=gen, device="cuda", dtype=torch.int32) for _ in range(2))
        near = torch.randint(-2 ** 63, 2 ** 63 - 1, (100,), generator=gen, device="cuda")
        for how in ({}, dict(window=5, sinks=1)):
            o = tree_attention(call.q, call.cache, call.table, call.lengths, call.offsets, DraftTree(positions, near, above), **how)
            assert torch.isfinite(o).all()


@pytest.mark.parametrize("batch", [3, 90])
def test_offsets_of_other_values_stay_inside(batch):
    """Offsets that do not ascend, lengths past the table: nothing outside is reached, and every call ends."""
    call = _Call((7,) * batch, (30,) * batch, 4, 2, 64, 16, BF16, 19, 2)
    gen = torch.Generator("cuda").manual_seed(2)
    for low, high in ((-5, 7 * batch + 5), (-2 ** 31, 2 ** 31 - 1)):
        offsets = torch.randint(low, high, (batch + 1,), generator=gen, device="cuda", dtype=torch.int32)
        lengths = torch.randint(low, high, (batch,), generator=gen, device="cuda", dtype=torch.int32)
        tree = draft_tree(call.parents, lengths, offsets)
        out = torch.zeros_like(call.q)
        tree_attention(call.q, call.cache, call.table, lengths, offsets, tree, out=out)
        uniforms = torch.rand(7 * batch, generator=gen, device="cuda")
        target = torch.rand((7 * batch, 50), generator=gen, device="cuda")
        kept = verify_drafts(target, None, torch.zeros_like(call.parents), call.parents, offsets, uniforms)
        keep_drafts(call.cache, call.table, lengths, offsets, kept.path, kept.counts)
        assert torch.isfinite(out).all() and all(torch.isfinite(t).all() for t in call.cache)


# ---- verification -------------------------------------------------------------


class _Drafts:
    def __init__(self, sizes, vocab, dtype, drawn, branch, seed, wide=True, before=0, behind=0, spread=2.0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.sizes, self.before = sizes, before
        rows = before + sum(sizes) + behind
        logits = torch.randn((rows, vocab), generator=gen, device="cuda") * spread
        self.target = logits.softmax(-1).to(dtype)
        near = logits + torch.randn((rows, vocab), generator=gen, device="cuda")
        self.draft = near.softmax(-1).to(dtype) if drawn else None
        self.trees = [make_tree(n, branch, seed + s) for s, n in enumerate(sizes)]
        self.parents, self.offsets = _packed(self.trees, before, behind), _offsets(sizes, before)
        # Drafts among the likeliest tokens, some of them twice behind the same one.
        self.tokens = torch.zeros(rows, dtype=torch.int64 if wide else torch.int32, device="cuda")
        at, weights = before, near.softmax(-1)
        for tree in self.trees:
            for j, p in enumerate(tree):
                if 0 <= p < j:
                    self.tokens[at + j] = weights[at + p].multinomial(1, generator=gen)[0]
            at += len(tree)
        self.uniforms = torch.rand(rows, generator=gen, device="cuda")

    def run(self):
        return verify_drafts(self.target, self.draft, self.tokens, self.parents, self.offsets, self.uniforms)

    def check(self, kept):
        target, draft = self.target.double().tolist(), None if self.draft is None else self.draft.double().tolist()
        tokens, uniforms, at = self.tokens.tolist(), self.uniforms.double().tolist(), self.before
        path, counts, after = kept.path.tolist(), kept.counts.tolist(), kept.next.tolist()
        assert all(x == -1 for x in path[:at])
        for b, tree in enumerate(self.trees):
            rows = slice(at, at + len(tree))
            if not tree:
                assert counts[b] == 0 and after[b] == -1
                continue
            want, token = verify(target[rows], None if draft is None else draft[rows], tokens[rows], tree, uniforms[rows])
            assert path[rows] == want + [-1] * (len(tree) - len(want)), b
            assert counts[b] == len(want) and after[b] == token, b
            at += len(tree)
        assert all(x == -1 for x in path[at:])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("sizes,vocab,branch", [
    ((1,), 1, 1), ((1, 2, 3), 2, 1), ((8,) * 40, 7, 1), ((8, 0, 20), 1023, 3), ((9,) * 6, 1024, 0), ((12, 30), 1025, 4),
    ((130, 70), 33, -1), ((200,), 9, 60), ((6, 6, 6), 5003, 2)])
def test_verify_drafts(dtype, drawn, sizes, vocab, branch):
    for seed in range(2):
        drafts = _Drafts(sizes, vocab, dtype, drawn, branch, 31 + seed, wide=seed == 0, before=3 * seed, behind=2 * seed)
        kept = drafts.run()
        assert kept.next.dtype == drafts.tokens.dtype
        drafts.check(kept)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_flat_probabilities(dtype, drawn):
    """Nearly equal weights, where a running sum in 32 bits would pass borders at other tokens; an odd vocabulary, rows
    that start anywhere."""
    drafts = _Drafts((5, 7, 1), 50257, dtype, drawn, 3, 77, spread=0.01)
    kept = drafts.run()
    drafts.check(kept)
    # Rows of wider tensors, from an odd place on.
    for name in ("target", "draft"):
        t = getattr(drafts, name)
        if t is not None:
            wide = torch.full((t.shape[0], t.shape[1] + 9), math.nan, dtype=t.dtype, device="cuda")
            wide[:, 3:-6] = t
            setattr(drafts, name, wide[:, 3:-6])
    for a, b in zip(kept, drafts.run()):
        assert torch.equal(a, b)


def test_verify_borders():
    """Numbers that reach a border exactly do not pass it."""
    target = torch.tensor([[0.25, 0.5, 0.25], [0.5, 0.25, 0.25]], device="cuda")
    draft = torch.tensor([[0.5, 0.25, 0.25], [0.25, 0.25, 0.5]], device="cuda")
    parents, offsets = _ints([-1, 0]), _ints([0, 2])

    def run(u0, u1, token, draft=draft):
        kept = verify_drafts(target, draft, _ints([0, token]), parents, offsets, torch.tensor([u0, u1], device="cuda"))
        return kept.counts.item(), kept.next.item()

    assert run(0.0, 0.5, 0) == (1, 1)             # 0.5 * 0.5 is not below 0.25; what is left: token 1 alone
    assert run(0.0, 0.5 - 2 ** -25, 0) == (2, 0)
    assert run(0.5, 0.0, 0) == (2, 1)             # a running sum of exactly 0.5 does not pass 0.5
    assert run(0.5 - 2 ** -25, 0.0, 0) == (2, 0)
    assert run(0.0, 0.25, 0, None) == (1, 1)
    assert run(0.75, 0.5, 1, None) == (1, 2) and run(0.25, 0.5, 1, None) == (1, 0) and run(0.5, 0.5, 1, None) == (1, 2)
    assert run(1.0, 0.0, 0) == (2, 2)             # outside of [0, 1): the last token that has a weight
    assert run(math.nan, math.nan, 0) == (1, 1) and run(-1.0, 0.0, 0) == (2, 0)


def test_verify_nothing_left():
    """The draft's probabilities cover the target's: a draft that is turned down all the same leaves them as they were."""
    target = torch.tensor([[0.25, 0.25, 0.5, 0.0]] * 3, device="cuda")
    draft = torch.tensor([[0.25, 0.25, 0.5, 1.0]] * 3, device="cuda")
    for tokens, want in (([0, 3, 3], ([0, -1, -1], 1, 2)), ([0, 3, 1], ([0, 2, -1], 2, 2))):
        kept = verify_drafts(target, draft, _ints(tokens), _ints([-1, 0, 0]), _ints([0, 3]), torch.full((3,), 0.5, device="cuda"))
        assert (kept.path.tolist(), kept.counts.item(), kept.next.item()) == want


def test_verify_odd_values():
    """NaN, infinite and negative probabilities count as 0, tokens outside the vocabulary are never kept, children
    whose parent does not come before them hang nowhere, and a token that is chosen twice has nothing left the second time."""
    for drawn in (True, False):
        drafts = _Drafts((12, 9, 30), 100, F32, drawn, 3, 5)
        drafts.target[::3, ::7] = math.nan
        drafts.target[1::3, 5::11] = -0.25
        drafts.target[2::5, 50] = math.inf
        if drawn:
            drafts.draft[::2, ::9] = math.nan
            drafts.draft[1::4, 1::5] = math.inf
        drafts.tokens[3::4] = torch.tensor([100, -1, 2 ** 40, -2 ** 63], device="cuda").repeat(4)[:drafts.tokens[3::4].shape[0]]
        drafts.check(drafts.run())
        drafts.target[:] = 0.0
        kept = drafts.run()
        assert kept.counts.tolist() == [1, 1, 1] and kept.next.tolist() == [-1, -1, -1]
    target = torch.tensor([[0.5, 0.5, 0.0]] * 4, device="cuda")
    kept = verify_drafts(target, None, _ints([0, 1, 1, 0]), _ints([-1, 0, 0, 0]), _ints([0, 4]),
                         torch.tensor([0.0, 0.75, 0.0, 0.5], device="cuda"))
    assert kept.path.tolist() == [0, 3, -1, -1] and kept.next.item() == 0


@pytest.mark.parametrize("drawn,branch", [(True, 1), (True, 3), (False, 3)])
def test_what_is_written_is_distributed_as_the_target_says(drawn, branch):
    """The token behind the first one, over 40,000 sequences: Pearson's chi squared with 6 degrees of freedom is above
    38.3 with a probability of 1e-6."""
    batch, n, vocab = 40000, 1 + 2 * branch, 7
    gen = torch.Generator("cuda").manual_seed(12)
    p, q = (torch.rand((1, vocab), generator=gen, device="cuda").add_(0.05) for _ in range(2))
    p, q = p / p.sum(), q / q.sum()
    parents = [-1] + [0] * branch + list(range(1, branch + 1))
    if drawn:
        tokens = q[0].multinomial(batch * n, replacement=True, generator=gen)
    else:  # the three likeliest of the draft
        first = q[0].topk(branch).indices
        tokens = torch.cat([first[:1], first, first]).repeat(batch)
    target, draft = p.expand(batch * n, vocab), q.expand(batch * n, vocab)
    assert target.stride(0) == 0
    kept = verify_drafts(target, draft if drawn else None, tokens, _ints(parents * batch), _ints(range(0, batch * n + 1, n)),
                         torch.rand(batch * n, generator=gen, device="cuda"))
    path = kept.path.reshape(batch, n)[:, 1].long()
    second = torch.where(kept.counts > 1, tokens.reshape(batch, n).gather(1, path.clamp_min(0)[:, None])[:, 0], kept.next)
    seen = torch.bincount(second, minlength=vocab).double()
    assert ((seen - batch * p[0].double()) ** 2 / (batch * p[0].double())).sum().item() < 38.3
    assert (kept.counts > 1).any() and (kept.counts == 1).any()


# ---- caches -------------------------------------------------------------------


def _layered(layers, pages, heads, page, dim, dtype, seed, token_major=False):
    caches = []
    for i in range(2):
        shape = (layers, pages, page, heads, dim) if token_major else (layers, pages, heads, page, dim)
        t = _rand(shape, dtype, seed + i)
        caches.append(t.transpose(2, 3) if token_major else t)
    return PagedCache(*caches)


@pytest.mark.parametrize("layers,heads,dim,page,token_major", [(1, 1, 64, 8, False), (3, 5, 128, 16, True), (2, 40, 64, 32, False)])
def test_keep_drafts(layers, heads, dim, page, token_major):
    new, cached = (1, 0, 7, 64, 300, 20), (5, 9, 0, 33, 100, 7)
    rng = random.Random(4)
    lengths = [n + c for n, c in zip(new, cached)]
    needed = [-(-length // page) for length in lengths]
    cache = _layered(layers, sum(needed) + 1, heads, page, dim, BF16, 1, token_major)
    order = list(range(sum(needed) + 1))
    rng.shuffle(order)
    rows = [[order.pop() for _ in range(count)] for count in needed]
    rows[5][-1] = -1  # some of the last sequence's rows are on no page
    table = _ints([row + [-1] * (max(needed) - len(row)) for row in rows])
    paths, counts = [], []
    for n in new:
        path = sorted(rng.sample(range(n), rng.randint(min(1, n), n)))
        counts.append(len(path))
        paths.append(path + [-1] * (n - len(path)))
    paths[3] = list(range(64))   # a chain that is kept whole
    counts[3] = 64
    counts[4] = 10 ** 6          # more than there are
    paths[4][5] = -3
    paths[4][6] = 300
    paths[4][7] = 2              # before its own place
    want = PagedCache(cache.k.clone(), cache.v.clone())
    for b, (n, length) in enumerate(zip(new, lengths)):
        moves = [(paths[b][j], j) for j in range(min(counts[b], n)) if j < paths[b][j] < n]
        for old, place in zip(cache, want):
            for source, j in moves:
                a, z = length - n + source, length - n + j
                if rows[b][a // page] >= 0 and rows[b][z // page] >= 0:
                    place[:, rows[b][z // page], :, z % page] = old[:, rows[b][a // page], :, a % page]
    path = _ints([p for its in paths for p in its])
    args = table, _ints(lengths), _offsets(new), path, _ints(counts)
    single = [PagedCache(cache.k[i].clone(), cache.v[i].clone()) for i in range(layers)]
    assert keep_drafts(cache, *args) is cache
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
    for i, one in enumerate(single):
        keep_drafts(one, *args)
        assert torch.equal(one.k, want.k[i]) and torch.equal(one.v, want.v[i])


def test_keep_drafts_before_the_cache():
    """Lengths below the new tokens: what would lie before the first place does not move."""
    cache = _layered(1, 2, 1, 8, 64, F16, 3)
    want = cache.k.clone()
    want[0, 0, :, 0] = cache.k[0, 0, :, 1]  # place 3 of six tokens, of which four are there, to place 2
    keep_drafts(cache, _ints([[0]]), _ints([4]), _ints([0, 6]), _ints([1, 2, 3, -1, -1, -1]), _ints([3]))
    assert torch.equal(cache.k, want)


@pytest.mark.parametrize("layers,pages,heads,page,dim,moves", [(1, 2, 1, 8, 64, 1), (3, 40, 5, 24, 128, 17), (2, 1300, 2, 8, 64, 600)])
@pytest.mark.parametrize("token_major", [False, True])
def test_copy_pages(layers, pages, heads, page, dim, moves, token_major):
    cache = _layered(layers, pages, heads, page, dim, F16, 2, token_major)
    order = list(range(pages))
    random.Random(moves).shuffle(order)
    to = order[:moves]
    pairs = [(random.Random(t).choice(order[moves:]), t) for t in to]  # some pages are copied more than once
    want = PagedCache(cache.k.clone(), cache.v.clone())
    for t in want:
        for a, b in pairs:
            t[:, b] = t[:, a]
    assert copy_pages(cache, pairs) is cache
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
    one = PagedCache(want.k[0], cache.v[layers - 1])  # one layer, keys and values from different tensors
    copy_pages(one, [])
    copy_pages(one, [(order[-1], to[0])])
    assert torch.equal(want.k[0, to[0]], want.k[0, order[-1]]) and torch.equal(cache.v[-1, to[0]], cache.v[-1, order[-1]])


def test_copy_pages_of_other_orders():
    """Keys with heads outside, values with tokens outside, both parts of something larger."""
    k = _rand((5, 3, 16, 128), BF16, 1)[..., :64]
    v = _rand((5, 16, 3, 64), BF16, 2).transpose(1, 2)
    before = k.clone(), v.clone()
    copy_pages(PagedCache(k, v), [(4, 0), (4, 1)])
    for t, old in zip((k, v), before):
        old[0] = old[1] = old[4].clone()
        assert torch.equal(t, old)


def test_pages_far_apart():
    """Offsets past 2^32 bytes: layers 5 GB apart, pages far into them."""
    pages = 40000
    k, v = (torch.zeros((2, pages, 4, 16, 512), dtype=BF16, device="cuda")[..., :64] for _ in range(2))
    cache = PagedCache(k, v)
    k[:, pages - 1] = 3.0
    v[:, pages - 1] = 5.0
    copy_pages(cache, [(pages - 1, pages - 2)])
    assert (k[:, pages - 2] == 3).all() and (v[:, pages - 2] == 5).all()
    k[1, pages - 1, :, 2] = 7.0
    keep_drafts(cache, _ints([[pages - 1]]), _ints([4]), _ints([0, 4]), _ints([0, 2, -1, -1]), _ints([2]))
    assert (k[1, pages - 1, :, 1] == 7).all() and (k[0, pages - 1, :, 1] == 3).all() and (k[:, pages - 3] == 0).all()
