"""Rotary positions, windowed attention and the paged cache on the GPU against
their plain forms in 64 bits."""
import math

import pytest
import torch

from ab_attention.streaming import PagedCache, append_cache, chunk_attention, rotary, window_attention
from streaming_reference import (HALF_STEP, attend, attend_grad, check_gradient, check_lse, check_output, logit_size,
                                 seen_mask, turned)

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, dtype, seed, scale=1.0, token_major=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    if token_major:
        b, h, n, d = shape
        return (torch.randn((b, n, h, d), generator=gen, device="cuda") * scale).to(dtype).transpose(1, 2)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


# ---- rotary -------------------------------------------------------------------


def _check_turned(got, x, ref):
    """One rounding of the result, and float32 sines (2^-22), products and sum of a pair of values."""
    u = HALF_STEP[x.dtype]
    size = x.double().abs().amax(-1, keepdim=True)
    assert ((got.double() - ref).abs() <= u * ref.abs() + 2.0 ** -20 * size + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("axes,dim,halves,joint", [((44, 42, 42), 128, False, False), ((32, 48, 48), 128, True, True),
                                                   ((16, 56, 56), 128, True, False), ((64,), 128, True, False),
                                                   ((10, 2, 4, 6), 24, False, False), ((2,), 8, False, True)])
@pytest.mark.parametrize("batch,heads,kv_heads,tokens", [(1, 1, 1, 1), (2, 5, 1, 37), (3, 12, 4, 260)])
def test_rotary(dtype, axes, dim, halves, joint, batch, heads, kv_heads, tokens):
    q = _rand((batch, heads, tokens, dim), dtype, 1)
    k = _rand((batch, kv_heads, tokens, dim), dtype, 2, token_major=True)
    gen = torch.Generator("cuda").manual_seed(3)
    pos = torch.randint(0, 200000, (batch, tokens, len(axes)), generator=gen, device="cuda")
    pairing = "halves" if halves else "adjacent"
    for p in (pos, pos[0].to(torch.int32), pos[0].float() / 8):
        a, b = rotary(q, k, p, axes, theta=1e4, pairing=pairing, joint=joint)
        assert b.stride() == k.stride()
        _check_turned(a, q, turned(q, p, axes, 1e4, halves, joint))
        _check_turned(b, k, turned(k, p, axes, 1e4, halves, joint))
    a, none = rotary(q, None, pos, axes, pairing=pairing, joint=joint)
    assert none is None
    _check_turned(a, q, turned(q, pos, axes, 1e4, halves, joint))


def test_rotary_reads_slices_and_leaves_the_rest():
    """Q and K as slices of one projection, and dims behind the axes bit for bit (infinities too)."""
    packed = _rand((2, 50, 3 * 4 * 128), BF16, 5)
    q, k, _ = (t.reshape(2, 50, 4, 128).transpose(1, 2) for t in packed.chunk(3, -1))
    q[..., 96:] = math.inf
    pos = torch.arange(50, device="cuda")[:, None].expand(50, 3)
    for pairing in ("adjacent", "halves"):
        a, b = rotary(q, k, pos, (32, 32, 32), pairing=pairing)
        assert torch.equal(a[..., 96:], q[..., 96:]) and torch.equal(b[..., 96:], k[..., 96:])
        _check_turned(a[..., :96], q[..., :96], turned(q[..., :96], pos, (32, 32, 32), halves=pairing == "halves"))
    q = _rand((1, 1, 3, 16), BF16, 6)
    q[..., 6:] = math.inf  # inside the unit of the last turned pair
    assert torch.equal(rotary(q, None, pos[:3, :1], (6,))[0][..., 6:], q[..., 6:])


def test_rotary_of_odd_places():
    """A tensor whose rows do not start on 16 bytes, one with its dims strided, none at all."""
    flat = _rand((2 * 3 * 40 + 1,), BF16, 7)
    q = flat[1:].reshape(1, 2, 3, 40)
    pos = torch.arange(3, device="cuda")[:, None]
    _check_turned(rotary(q, None, pos, (40,))[0], q, turned(q, pos, (40,)))
    q = _rand((1, 2, 40, 3), BF16, 8).transpose(2, 3)
    _check_turned(rotary(q, None, pos, (40,))[0], q, turned(q, pos, (40,)))
    empty = torch.empty((2, 3, 0, 64), dtype=BF16, device="cuda")
    assert rotary(empty, empty, torch.empty((0, 1), dtype=torch.int32, device="cuda"), (64,))[0].shape == empty.shape


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary_gradient(dtype):
    """The gradient is the opposite rotation; and the rotation of it gives it back."""
    q, k = _rand((2, 6, 45, 128), dtype, 1).requires_grad_(), _rand((2, 2, 45, 128), dtype, 2).requires_grad_()
    dq, dk = _rand((2, 6, 45, 128), dtype, 3, token_major=True), _rand((2, 2, 45, 128), dtype, 4)
    pos = torch.randint(0, 1000, (45, 3), device="cuda")
    axes = (44, 42, 42)
    a, b = rotary(q, k, pos, axes)
    gq, gk = torch.autograd.grad((a, b), (q, k), (dq, dk), retain_graph=True)
    _check_turned(gq, dq, turned(dq, pos, axes, inverse=True))
    _check_turned(gk, dk, turned(dk, pos, axes, inverse=True))
    assert torch.equal(torch.autograd.grad(b, k, dk, retain_graph=True)[0], gk)
    assert torch.equal(torch.autograd.grad(a, q, dq)[0], gq)
    assert torch.equal(torch.autograd.grad(rotary(q, None, pos, axes)[0], q, dq)[0], gq)


# ---- window attention ---------------------------------------------------------


def _window_case(batch, heads, kv_heads, tokens, dim, dtype, window, sinks, frame, lengths=None, token_major=False, seed=0,
                 junk=None, scale=None):
    q = _rand((batch, heads, tokens, dim), dtype, seed + 1, 2.0, token_major)
    k = _rand((batch, kv_heads, tokens, dim), dtype, seed + 2, 1.0, token_major)
    v = _rand((batch, kv_heads, tokens, dim), dtype, seed + 3, 1.0, token_major)
    if junk is not None:  # what lies in the padding is nobody's business
        for b, length in enumerate(lengths):
            for t in (q, k, v):
                t[b, :, length:] = junk
    dev_lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = window_attention(q, k, v, window=window, sinks=sinks, frame=frame, lengths=dev_lengths, scale=scale,
                                return_lse=True)
    assert out.stride() == q.stride() and out.dtype == dtype
    at = torch.arange(tokens, device="cuda")
    for b in range(batch):
        n = tokens if lengths is None else max(0, min(lengths[b], tokens))
        mask = seen_mask(at, at, window, sinks, frame) & (at[:, None] < n) & (at[None] < n)
        o, l, spread = attend(torch.nan_to_num(q[b], 0, 0, 0), k[b], v[b], mask, scale)
        check_output(out[b], o, spread, dtype)
        check_lse(lse[b], l, dim, logit_size(q[b, :, :n], k[b, :, :n], scale))
        assert (out[b, :, n:] == 0).all() and (lse[b, :, n:] == -math.inf).all()
    same = window_attention(q, k, v, window=window, sinks=sinks, frame=frame, lengths=dev_lengths, scale=scale)
    assert torch.equal(same, out)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 7, 31, 32, 33, 63, 65, 127, 128, 129, 300])
def test_window_lengths(tokens, dim, dtype):
    _window_case(1, 2, 1, tokens, dim, dtype, 40, 3, 1, seed=tokens)


@pytest.mark.parametrize("window,sinks,frame", [(None, 0, 1), (1, 0, 1), (1, 1, 1), (2, 5, 1), (33, 0, 1), (64, 40, 1),
                                                (200, 150, 1), (10000, 3, 1), (100, 10000, 1), (None, 0, 7), (1, 0, 100),
                                                (2, 1, 31), (3, 2, 37), (1, 3, 130), (2, 1, 260), (1, 0, 5000),
                                                (2 ** 40, 2 ** 40, 1), (1, 0, 2 ** 40), (2 ** 31, 7, 3)])
def test_window_masks(window, sinks, frame):
    _window_case(2, 3, 3, 517, 128, BF16, window, sinks, frame)


@pytest.mark.parametrize("heads,kv_heads,token_major", [(8, 2, False), (6, 1, True), (4, 4, True)])
def test_window_heads_and_strides(heads, kv_heads, token_major):
    _window_case(2, heads, kv_heads, 333, 128, BF16, 100, 4, 1, token_major=token_major)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("junk", [math.nan, math.inf])
def test_window_padded_batch(dim, junk):
    _window_case(5, 4, 2, 200, dim, BF16, 50, 2, 1, lengths=[200, 0, 1, 77, 129], junk=junk)
    _window_case(2, 2, 2, 200, dim, F16, 2, 1, 48, lengths=[31, 150], junk=junk)


def test_window_lengths_outside():
    """Lengths below zero are zero, those above the tokens are the tokens."""
    _window_case(3, 2, 2, 70, 64, BF16, 20, 0, 1, lengths=[-5, 1000, 70])


def test_window_scale():
    _window_case(1, 2, 2, 150, 128, BF16, None, 0, 1, scale=0.02)
    _window_case(1, 2, 2, 150, 128, BF16, None, 0, 1, scale=-0.05)
    _window_case(1, 2, 2, 150, 128, BF16, 30, 0, 1, scale=0.0)


def test_window_many_tiles():
    """More than 64 tiles of rows: the order of the XCDs' shares."""
    _window_case(1, 3, 1, 8500, 64, BF16, 300, 5, 1)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_window_values_that_are_not_finite_reach_only_who_sees_them(value):
    """Token 100's value row: queries before it, and those whose window has passed it, do not change."""
    shape = (1, 2, 300, 128)
    q, k, v = (_rand(shape, BF16, s) for s in (1, 2, 3))
    how = dict(window=40, sinks=2)
    clean = window_attention(q, k, v, **how)
    v[:, :, 100, 5] = value
    got = window_attention(q, k, v, **how)
    hit = torch.zeros(300, dtype=torch.bool, device="cuda")
    hit[100:140] = True
    assert torch.equal(got[:, :, ~hit], clean[:, :, ~hit])
    assert torch.equal(got[:, :, hit][..., :5], clean[:, :, hit][..., :5])
    bad = got[:, :, hit][..., 5]
    assert bad.isnan().all() if math.isnan(value) else (bad == value).all()
    # A key row: nobody before it, nobody behind its window.
    v[:, :, 100, 5] = 0
    k[:, :, 100] = value if not math.isinf(value) else math.nan
    got = window_attention(q, k, v, **how)
    v_clean = window_attention(q, torch.nan_to_num(k), v, **how)
    assert torch.equal(got[:, :, ~hit], v_clean[:, :, ~hit])


def test_window_large_logits():
    """The reference moves with the maximum: logits of hundreds, rising and falling along the keys."""
    n = 400
    q, k, v = (_rand((1, 1, n, 128), BF16, s) for s in (1, 2, 3))
    for ramp in (torch.linspace(0, 60, n), torch.linspace(60, 0, n)):
        big = (k.float() + q.float().mean(2, keepdim=True) + ramp.cuda()[None, None, :, None] * 0.2).to(BF16)
        out, lse = window_attention(q, big, v, return_lse=True)
        at = torch.arange(n, device="cuda")
        o, l, spread = attend(q[0], big[0], v[0], seen_mask(at, at, None, 0, 1))
        check_lse(lse[0], l, 128, logit_size(q, big))
        # Logits are off by up to their size times 2^-24 * 128; the weights by as much.
        u = HALF_STEP[BF16]
        room = (u * (1 + u) + logit_size(q, big) * 128 * 2.0 ** -24 * 2) * (spread + o.abs()) + 1e-4
        assert ((out[0].double() - o).abs() <= room).all()


@pytest.mark.parametrize("heads,tokens", [(3, 1), (1, 900), (700, 40)])
def test_window_odd_grids(heads, tokens):
    """One row in all, one head of several tiles, more heads than tiles."""
    _window_case(1, heads, heads, tokens, 64, BF16, 100, 1, 1)


def test_window_of_no_tokens():
    empty = torch.empty((2, 3, 0, 64), dtype=BF16, device="cuda")
    out, lse = window_attention(empty, empty, empty, window=3, return_lse=True)
    assert out.shape == empty.shape and lse.shape == (2, 3, 0)
    none = torch.empty((0, 3, 5, 64), dtype=BF16, device="cuda")
    assert window_attention(none, none, none).shape == none.shape


def _grad_case(batch, heads, kv_heads, tokens, dim, dtype, window, sinks, frame, lengths=None, token_major=False, seed=0,
               with_lse=False, scale=None, junk=None):
    q = _rand((batch, heads, tokens, dim), dtype, seed + 1, 1.5, token_major)
    k = _rand((batch, kv_heads, tokens, dim), dtype, seed + 2, 1.0, token_major)
    v = _rand((batch, kv_heads, tokens, dim), dtype, seed + 3, 1.0, not token_major)
    do = _rand((batch, heads, tokens, dim), dtype, seed + 4, 1.0, token_major)
    dlse = _rand((batch, heads, tokens), F32, seed + 5) if with_lse else None
    n_of = [tokens if lengths is None else max(0, min(n, tokens)) for n in (lengths or [0] * batch)]
    if junk is not None:
        for b, n in enumerate(n_of):
            for t in (q, k, v, do):
                t[b, :, n:] = junk
    for t in (q, k, v):
        t.requires_grad_()
    dev_lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = window_attention(q, k, v, window=window, sinks=sinks, frame=frame, lengths=dev_lengths, scale=scale,
                                return_lse=True)
    if with_lse:
        grads = torch.autograd.grad((out, lse), (q, k, v), (do, dlse), retain_graph=True)
        again = torch.autograd.grad((out, lse), (q, k, v), (do, dlse))
    else:
        grads = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
        again = torch.autograd.grad(out, (q, k, v), do)
    at = torch.arange(tokens, device="cuda")
    for b, n in enumerate(n_of):
        want, room = attend_grad(q[b, :, :n], k[b, :, :n], v[b, :, :n], do[b, :, :n],
                                 seen_mask(at[:n], at[:n], window, sinks, frame), None if dlse is None else dlse[b, :, :n], scale)
        for name, got, w, r in zip("qkv", grads, want, room):
            check_gradient(got[b, :, :n], w, r, dtype, name)
            assert (got[b, :, n:] == 0).all(), name
    for t, g, a in zip((q, k, v), grads, again):
        assert g.shape == t.shape and g.dtype == t.dtype and g.stride() == t.stride()
        assert torch.equal(g, a)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 64, 127, 129, 300])
def test_window_gradient_lengths(tokens, dim, dtype):
    _grad_case(1, 2, 1, tokens, dim, dtype, 40, 3, 1, seed=tokens)


@pytest.mark.parametrize("window,sinks,frame", [(None, 0, 1), (1, 0, 1), (2, 5, 1), (33, 0, 1), (64, 40, 1), (20, 300, 1),
                                                (10000, 3, 1), (None, 0, 7), (1, 0, 100), (2, 1, 31), (3, 2, 37), (1, 3, 130),
                                                (2, 1, 260), (1, 0, 5000), (2 ** 40, 2 ** 40, 1), (1, 1, 129)])
def test_window_gradient_masks(window, sinks, frame):
    _grad_case(2, 3, 3, 517, 128, BF16, window, sinks, frame)


@pytest.mark.parametrize("heads,kv_heads,window,sinks", [(2, 2, 400, 1000), (4, 1, 90, 900), (4, 1, 90, 870)])
def test_window_gradient_sinks_in_all_tiles(heads, kv_heads, window, sinks):
    """The sinks reach into the last tile of keys (or the one before it), and behind it."""
    _grad_case(1, heads, kv_heads, 1000, 64, BF16, window, sinks, 1)


@pytest.mark.parametrize("heads,kv_heads,token_major", [(8, 2, False), (6, 1, True), (4, 4, True)])
def test_window_gradient_heads_and_strides(heads, kv_heads, token_major):
    _grad_case(2, heads, kv_heads, 333, 128, BF16, 60, 4, 1, token_major=token_major, with_lse=True)


@pytest.mark.parametrize("dim", [64, 128])
def test_window_gradient_padded_batch(dim):
    for junk in (math.nan, math.inf):
        _grad_case(5, 4, 2, 200, dim, BF16, 50, 2, 1, lengths=[200, 0, 1, 77, 129], junk=junk)
        _grad_case(2, 2, 1, 400, dim, F16, 2, 1, 48, lengths=[31, 350], junk=junk, with_lse=True)


def test_window_gradient_many_tiles_and_scale():
    _grad_case(1, 3, 1, 8500, 64, BF16, 300, 5, 1)
    _grad_case(1, 2, 2, 200, 128, BF16, 50, 0, 1, scale=-0.06)


@pytest.mark.parametrize("tokens,stride", [(100000, 20480), (110000, 20480)])
def test_window_rows_4_gib_apart(tokens, stride):
    """A head whose rows span almost 4 GiB is read in place, a longer one from a copy: the bits of contiguous tensors."""
    base = torch.empty(tokens * stride, dtype=BF16, device="cuda")
    views = [base.as_strided((1, 1, tokens, 64), (0, 0, stride, 1), 64 * i) for i in range(4)]
    for i, view in enumerate(views):
        view.copy_(_rand((1, 1, tokens, 64), BF16, i + 1))
    leaves = [t.detach().requires_grad_() for t in views[:3]]
    plain = [t.detach().contiguous().requires_grad_() for t in views[:3]]
    out, want = (window_attention(*t, window=300, sinks=3) for t in (leaves, plain))
    assert torch.equal(out, want)
    for g, w in zip(torch.autograd.grad(out, leaves, views[3]), torch.autograd.grad(want, plain, views[3].contiguous())):
        assert torch.equal(g, w)


def test_window_gradient_parts_of_the_graph():
    """Only some of q, k, v, only the normaliser, an expanded gradient, a value shared by q and k."""
    q, k, v = (_rand((1, 2, 90, 64), BF16, s) for s in (1, 2, 3))
    how = dict(window=30, sinks=1, return_lse=True)
    ones = torch.ones((), dtype=BF16, device="cuda").expand(1, 2, 90, 64)
    full = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(window_attention(*full, **how)[0], full, ones.contiguous())
    got = torch.autograd.grad(window_attention(*full, **how)[0], full, ones)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = k.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(window_attention(q, one, v, **how)[0], one, ones)[0], want[1])
    lse = window_attention(*full, **how)[1]
    dq, dk = torch.autograd.grad(lse.sum(), full[:2])
    at = torch.arange(90, device="cuda")
    (wq, wk, _), (rq, rk, _) = attend_grad(q[0], k[0], v[0], torch.zeros_like(q[0]), seen_mask(at, at, 30, 1, 1),
                                           torch.ones_like(lse[0]))
    check_gradient(dq[0], wq, rq, BF16)
    check_gradient(dk[0], wk, rk, BF16)
    same = q.clone().requires_grad_()
    both = torch.autograd.grad(window_attention(same, same, v, **how)[0], same, ones)[0]
    pair = [q.clone().requires_grad_() for _ in range(2)]
    dq, dk = torch.autograd.grad(window_attention(*pair, v, **how)[0], pair, ones)
    assert torch.equal(both, dq + dk)


def test_window_gradient_without_the_rest():
    """The C entry with out alone: within the room that the output's rounding is given, and no nearer than with both."""
    from ab_attention import _lib
    from ab_attention import streaming as st

    shape = (1, 2, 300, 64)
    q, k, v, do = (_rand(shape, BF16, s) for s in (1, 2, 3, 4))
    how = (50, 3, 1, 64 ** -0.5)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out, lse = window_attention(*leaves, window=50, sinks=3, return_lse=True)
    with_rest = torch.autograd.grad(out, leaves, do)
    grads = [torch.empty_like(q) for _ in range(3)]
    behind = st._GRAD_REST.pack(do.data_ptr(), 0, *(g.data_ptr() for g in grads), *do.stride()[:3],
                                *(s for g in grads for s in g.stride()[:3]))
    args = (q, k, v, out.detach(), None, lse.detach(), None, *how)
    size = _lib.raw("ab_window_grad_workspace_bytes")(st._window_args(*args) + behind)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    st._call("ab_window_attention_grad", q.device, st._window_args(*args, workspace.data_ptr(), size) + behind)
    at = torch.arange(300, device="cuda")
    want, room = attend_grad(q[0], k[0], v[0], do[0], seen_mask(at, at, 50, 3, 1))
    for g, both, w, r in zip(grads, with_rest, want, room):
        check_gradient(g[0], w, r, BF16)
        assert (both[0].double() - w).norm() <= 1.001 * (g[0].double() - w).norm()


def test_window_gradient_of_small_probabilities():
    """fp16 keys that every query gives about 2^-18, where fp16 itself has a quarter of its bits: dV rounds them
    relative to their size all the same."""
    n, dim = 1000, 64
    q, k, v, do = (_rand((1, 1, n, dim), F16, s) for s in (1, 2, 3, 4))
    q[..., 0], k[..., 0] = 4, 0
    k[:, :, 0] = 0
    k[:, :, 0, 0] = 25  # 25 * 4 / 8 * log2(e): 18 above the others
    do *= 32
    leaf = v.clone().requires_grad_()
    dv = torch.autograd.grad(window_attention(q, k, leaf), leaf, do)[0][0].double()
    at = torch.arange(n, device="cuda")
    mask = seen_mask(at, at, None, 0, 1)
    (_, _, want), _ = attend_grad(q[0], k[0], v[0], do[0], mask)
    p = torch.softmax((q[0].double() @ k[0].double().transpose(1, 2) / 8).masked_fill(~mask, -math.inf), -1)
    # Every P rounded once with a sign of its own (a half step bounds the deviation), and the gradient once.
    u = HALF_STEP[F16]
    room = u * (p.transpose(1, 2) ** 2 @ do[0].double() ** 2)[:, 1:].sum().sqrt() + u * want[:, 1:].norm() + 2.0 ** -25 * (n * dim) ** 0.5
    assert (dv - want)[:, 1:].norm() <= room


def test_window_gradient_against_differences():
    """A directional derivative of a weighted sum of the output and the normaliser in 64 bits, by central differences of
    the definition, against the kernels' gradients."""
    shape, n = (1, 2, 140, 64), 140
    q, k, v, do = (_rand(shape, F16, s).requires_grad_(s < 4) for s in (1, 2, 3, 4))
    how = dict(window=50, sinks=3)
    at = torch.arange(n, device="cuda")
    mask = seen_mask(at, at, 50, 3, 1)
    grads = torch.autograd.grad(window_attention(q, k, v, **how), (q, k, v), do)

    def loss(*t):
        return (attend(*(x.double()[0] for x in t), mask)[0] * do[0].double()).sum().item()

    for i, name in enumerate("qkv"):
        step = _rand(shape, F32, 10 + i).double()
        sides = [[t.detach().double() + (e * step if j == i else 0) for j, t in enumerate((q, k, v))] for e in (1e-5, -1e-5)]
        slope = (loss(*sides[0]) - loss(*sides[1])) / 2e-5
        got = (grads[i].double() * step).sum().item()
        # Each value of the gradient carries a few roundings of 2^-11 with signs of their own: five of their standard deviations.
        assert abs(got - slope) <= 5 * 4 * 2.0 ** -11 * (grads[i].double() * step).norm().item() + 1e-4 * abs(slope), (name, got, slope)


# ---- paged cache and chunks ---------------------------------------------------


def _cache(new, total, heads, dim, page, dtype, seed=0, spare=2, token_major=False):
    """(cache, table on the host, lengths, offsets) with all pages filled at random."""
    gen = torch.Generator().manual_seed(seed)
    needed = [-(-t // page) for t in total]
    pages = sum(needed) + spare
    shape = (pages, heads, page, dim)
    cache = PagedCache(*(_rand(shape, dtype, seed + s, 1.0, token_major) for s in (11, 12)))
    table = torch.full((len(total), max(needed + [1])), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=gen), 0
    for b, n in enumerate(needed):
        table[b, :n] = order[at:at + n]
        at += n
    offsets = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return cache, table, torch.tensor(total, dtype=torch.int32), offsets


def _check_chunk(out, lse, q, cache, table, total, offsets, window, sinks, frame, dtype):
    page, pages = cache.k.shape[2], cache.k.shape[0]
    for b, length in enumerate(total.tolist()):
        start, stop = offsets[b].item(), offsets[b + 1].item()
        if stop == start:
            continue
        keys = torch.arange(max(0, min(length, table.shape[1] * page)), device="cuda")
        at = table[b].cuda().long()[keys // page]
        there = (at >= 0) & (at < pages)
        mask = seen_mask(length - (stop - start) + torch.arange(stop - start, device="cuda"), keys, window, sinks, frame)
        at = at.clamp(0, pages - 1)
        k, v = (t[at, :, keys % page].transpose(0, 1) for t in cache)
        qb = q[start:stop].transpose(0, 1)
        o, l, spread = attend(qb, k, v, mask & there)
        check_output(out[start:stop].transpose(0, 1), o, spread, dtype)
        check_lse(lse[start:stop].transpose(0, 1), l, q.shape[-1], logit_size(qb, k))


def _chunk_case(new, total, heads, kv_heads, dim, page, dtype=BF16, window=None, sinks=0, frame=1, evict=False, seed=0,
                token_major=False):
    cache, table, lengths, offsets = _cache(new, total, kv_heads, dim, page, dtype, seed, token_major=token_major)
    tokens = int(offsets[-1])
    q = _rand((tokens + 5, heads, dim), dtype, seed + 1, 2.0)
    for b, (n, length) in enumerate(zip(new, total)):
        # Behind the last token a page holds whatever was there.
        if length % page:
            for t in cache:
                t[table[b, length // page].long(), :, length % page:] = math.nan
        if evict and window is not None:
            low = max(0, (length - n) // frame - window + 1) * frame
            gone = slice(-(-min(sinks * frame, low) // page), low // page)
            for t in cache:
                t[table[b, gone].long()] = math.nan
            table[b, gone] = -1 if b % 2 else 2 ** 31 - 1
    out = torch.full((tokens + 5, heads, dim), 7.0, dtype=dtype, device="cuda")
    dev = [t.cuda() for t in (table, lengths, offsets)]
    got, lse = chunk_attention(q, cache, *dev, window=window, sinks=sinks, frame=frame, return_lse=True, out=out)
    assert got is out and (out[tokens:] == 7).all()
    _check_chunk(out, lse, q, cache, table, lengths, offsets, window, sinks, frame, dtype)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("page", [8, 24, 32, 64, 1560])
def test_chunk_pages(dim, dtype, page):
    _chunk_case([1, 5, 64, 1, 200], [1, 5, 300, 1000, 333], 4, 2, dim, page, dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (12, 4), (40, 8)])
def test_chunk_single_tokens(heads, kv_heads):
    """One token in each sequence, from the first one to long caches: split over workgroups."""
    _chunk_case([1] * 6, [1, 2, 33, 700, 4097, 20000], heads, kv_heads, 128, 64)


@pytest.mark.parametrize("window,sinks,frame", [(1, 0, 1), (50, 0, 1), (64, 4, 1), (300, 100, 1), (2, 1, 48), (1, 1, 100),
                                                (3, 0, 7)])
@pytest.mark.parametrize("new,total", [([1, 3, 150, 96], [900, 700, 150, 530]), ([1, 1], [5000, 130])])
def test_chunk_windows(window, sinks, frame, new, total):
    """Pages that nobody sees any more are given back, and hold NaN."""
    _chunk_case(new, total, 6, 2, 128, 32, window=window, sinks=sinks, frame=frame, evict=True)


def test_chunk_empty_sequences():
    _chunk_case([0, 3, 0, 0, 1, 0], [10, 40, 0, 70, 1, 5], 4, 4, 64, 16)
    _chunk_case([0], [100], 2, 1, 64, 16)


def test_chunk_token_major_cache():
    _chunk_case([5, 1, 140], [100, 64, 777], 8, 4, 128, 16, token_major=True)


def test_chunk_many_sequences():
    """More sequences than lanes of a wave."""
    new = [(7 * b) % 4 for b in range(150)]
    _chunk_case(new, [n + (13 * b) % 90 for b, n in enumerate(new)], 2, 1, 64, 16)


def test_chunk_holes():
    """Pages missing in the middle, all of a sequence's pages missing, more new tokens than the length says."""
    cache, table, lengths, offsets = _cache([4, 2, 9, 1], [300, 100, 64, 2000], 2, 128, 16, BF16)
    table[0, 3:7] = -1
    table[0, 18] = 10 ** 6
    table[1] = -1
    table[3, 20:100] = -7
    lengths[2] = 5  # positions -4 .. 4: the first four queries see nothing
    q = _rand((16, 4, 128), BF16, 3, 2.0)
    for window, sinks in ((None, 0), (40, 8)):
        out, lse = chunk_attention(q, cache, table.cuda(), lengths.cuda(), offsets.cuda(), window=window, sinks=sinks, return_lse=True)
        _check_chunk(out, lse, q, cache, table, lengths, offsets, window, sinks, 1, BF16)
        assert (out[4:6] == 0).all() and (lse[4:6] == -math.inf).all() and (out[6:10] == 0).all()


def test_chunk_bounds_of_device_sizes():
    """Lengths beyond the table, offsets beyond the tokens: what is there is done, nothing else is touched."""
    cache, table, lengths, offsets = _cache([2, 2], [64, 64], 1, 64, 16, BF16)
    q = _rand((4, 1, 64), BF16, 3)
    many = torch.tensor([10 ** 6, 64], dtype=torch.int32)
    out, lse = chunk_attention(q, cache, table.cuda(), many.cuda(), offsets.cuda(), return_lse=True)
    _check_chunk(out, lse, q, cache, table, torch.tensor([64, 64]), offsets, None, 0, 1, BF16)
    far = torch.tensor([0, 2, 1000], dtype=torch.int32)
    chunk_attention(q, cache, table.cuda(), lengths.cuda(), far.cuda(), out=out)
    back = torch.tensor([3, 1, -5], dtype=torch.int32)
    out.fill_(3)
    chunk_attention(q, cache, table.cuda(), lengths.cuda(), back.cuda(), out=out)
    assert (out == 3).all()


def test_chunk_and_window_rest_of_the_output():
    """The C entries with out_rest: the same output, and together with the rest nearer to the definition. A query of
    one key's weight alone has just that key's value."""
    from ab_attention import _lib
    from ab_attention import streaming as st

    tokens, heads, dim = 700, 3, 64
    q, k, v = (_rand((1, heads, tokens, dim), BF16, s, 2.0 if s == 1 else 1.0) for s in (1, 2, 3))
    how = (300, 4, 1, dim ** -0.5)
    rest = torch.empty_like(q)
    out, _ = st._window_forward(q, k, v, None, *how, False, rest)
    assert torch.equal(out, window_attention(q, k, v, window=300, sinks=4))
    assert torch.equal(out, window_attention(q, k, v.clone().requires_grad_(), window=300, sinks=4))
    at = torch.arange(tokens, device="cuda")
    o, _, _ = attend(q[0], k[0], v[0], seen_mask(at, at, 300, 4, 1))
    both = out[0].double() + rest[0].double()
    assert (both - o).norm() < 0.9 * (out[0].double() - o).norm()
    assert torch.equal(both[:, 0], v[0, :, 0].double())

    few = [t[:, :1, :140].contiguous() for t in (q, k, v)]  # so few rows that their keys are split
    rest = torch.empty_like(few[0])
    packed = st._window_args(*few, rest, rest, None, None, 0, 0, 1, dim ** -0.5)
    out, _ = st._window_forward(*few, None, 0, 0, 1, dim ** -0.5, False, rest)
    assert torch.equal(out, window_attention(*few)) and _lib.raw("ab_window_workspace_bytes")(packed) % (dim * 4 + 12) == 0
    o, _, _ = attend(*(t[0] for t in few), seen_mask(at[:140], at[:140], None, 0, 1))
    both = out[0].double() + rest[0].double()
    assert (both - o).norm() < 0.9 * (out[0].double() - o).norm()
    assert torch.equal(both[:, 0], few[2][0, :, 0].double())

    cache, table, lengths, offsets = _cache([5, 1], [130, 4000], heads, dim, 16, BF16)
    q = _rand((6, heads, dim), BF16, 5, 2.0)
    want = chunk_attention(q, cache, table.cuda(), lengths.cuda(), offsets.cuda())
    dev = [t.cuda() for t in (lengths, offsets, table)]
    out, rest = torch.empty_like(q), torch.full_like(q, 9.0)
    for size in (0, 1 << 24):  # whole rows, rows in parts
        workspace = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        packed = st._WINDOW.pack(q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), out.data_ptr(), rest.data_ptr(), 0,
                                 *(t.data_ptr() for t in dev), 2, heads, heads, 6, dim, 0, cache.k.shape[0], 16, table.shape[1],
                                 0, 0, 1, dim ** -0.5, 0, q.stride(1), q.stride(0), *cache.k.stride()[:3],
                                 *cache.v.stride()[:3], 0, out.stride(1), out.stride(0), workspace.data_ptr() if size else 0, size)
        assert _lib.raw("ab_window_workspace_bytes")(packed) <= 1 << 24
        st._call("ab_chunk_attention", q.device, packed)
        # What rounding the output took is at most half a step of it, and what is left of that its own rounding.
        assert (rest.double().abs() <= 2.0 ** -8 * out.double().abs() + 1e-6).all()
    assert torch.equal(out, want)


def test_chunk_and_append_refuse_rows_that_share_memory():
    cache, *where = _cache([4], [40], 2, 64, 16, BF16)
    where = [t.cuda() for t in where]
    x = _rand((4, 2, 64), BF16, 1)
    with pytest.raises(ValueError, match="each its own"):
        chunk_attention(x, cache, *where, out=x[:1].expand(4, 2, 64))
    wide = PagedCache(cache.k, cache.v[:1].expand(cache.k.shape))
    chunk_attention(x, wide, *where)  # may be read
    with pytest.raises(ValueError, match="expanded"):
        append_cache(wide, x, x, *where)


def test_chunk_of_many_sequences_in_no_order():
    """Offsets that go back and forth over more sequences than lanes of a wave: rows and pages that are no sequence's
    stay as they were."""
    batch, tokens, heads = 70, 100, 8
    cache, table, lengths, _ = _cache([1] * batch, [64] * batch, 1, 64, 16, BF16)
    offsets = torch.zeros(batch + 1, dtype=torch.int32)
    offsets[:2] = torch.tensor([50, 100])
    guard = torch.full((tokens + 400, heads, 64), 3.0, dtype=BF16, device="cuda")
    q = _rand((tokens + 400, heads, 64), BF16, 3)[200:200 + tokens]
    chunk_attention(q, cache, table.cuda(), lengths.cuda(), offsets.cuda(), out=guard[200:200 + tokens])
    assert (guard[:250] == 3).all() and (guard[200 + tokens:] == 3).all()


def test_chunk_of_nothing():
    cache, table, lengths, offsets = (t.cuda() if torch.is_tensor(t) else t for t in _cache([1], [9], 2, 64, 16, BF16))
    q = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    assert chunk_attention(q, cache, table, lengths, offsets).shape == q.shape
    bare = PagedCache(*(t[:0] for t in cache))
    out, lse = chunk_attention(_rand((1, 2, 64), BF16, 1), bare, table, lengths, offsets, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = chunk_attention(_rand((1, 2, 64), BF16, 1), cache, table[:, :0], lengths, offsets, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_append_and_the_far_end_of_a_cache():
    """Pages past 2^32 bytes of a cache, written and read."""
    pages, page, heads, dim = 4400, 64, 64, 128  # 4.6 GB each
    cache = PagedCache(*(torch.empty((pages, heads, page, dim), dtype=BF16, device="cuda") for _ in range(2)))
    table = torch.tensor([[4399, 7, 4398]], dtype=torch.int32)
    lengths, offsets = torch.tensor([150], dtype=torch.int32), torch.tensor([0, 150], dtype=torch.int32)
    k, v, q = (_rand((150, heads, dim), BF16, s) for s in (1, 2, 3))
    dev = [t.cuda() for t in (table, lengths, offsets)]
    append_cache(cache, k, v, *dev)
    assert torch.equal(cache.k[4398, :, :22], k[128:].transpose(0, 1)) and torch.equal(cache.v[4399], v[:64].transpose(0, 1))
    out, lse = chunk_attention(q, cache, *dev, return_lse=True)
    _check_chunk(out, lse, q, cache, table, lengths, offsets, None, 0, 1, BF16)


@pytest.mark.parametrize("dim,heads,page", [(64, 1, 8), (128, 5, 64), (64, 8, 1560)])
@pytest.mark.parametrize("token_major", [False, True])
def test_append(dim, heads, page, token_major):
    new, total = [1, 0, 70, 3, 9], [1, 50, 200, 1600, 9]
    cache, table, lengths, offsets = _cache(new, total, heads, dim, page, F16, token_major=token_major)
    table[3, 0] = -1  # not written to: its new tokens lie behind
    k = _rand((90, heads, dim), F16, 5)
    v = _rand((90, 3, heads, dim), F16, 6)[:, 1]  # a slice of a projection
    want = PagedCache(cache.k.clone(), cache.v.clone())
    for b, (n, length) in enumerate(zip(new, total)):
        for i in range(n):
            at = length - n + i
            for dst, src in zip(want, (k, v)):
                dst[table[b, at // page].long(), :, at % page] = src[offsets[b] + i]
    assert append_cache(cache, k, v, table.cuda(), lengths.cuda(), offsets.cuda()) is cache
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)


def test_chunk_without_a_window_over_a_long_cache():
    """Positions past 100,000, pages in any order, a prompt and a token."""
    _chunk_case([130, 1], [100100, 120001], 2, 1, 64, 256)


def test_append_drops_what_has_no_place():
    cache, table, lengths, offsets = _cache([4, 4, 4], [4, 40, 4], 2, 64, 16, BF16)
    before = PagedCache(cache.k.clone(), cache.v.clone())
    table[0, 0] = -1
    lengths[1] = 1000  # past the table
    lengths[2] = 2     # two of four rows lie before position 0
    k, v = _rand((12, 2, 64), BF16, 1), _rand((12, 2, 64), BF16, 2)
    append_cache(cache, k, v, table.cuda(), lengths.cuda(), offsets.cuda())
    before.k[table[2, 0].long(), :, :2] = k[10:].transpose(0, 1)
    before.v[table[2, 0].long(), :, :2] = v[10:].transpose(0, 1)
    assert torch.equal(cache.k, before.k) and torch.equal(cache.v, before.v)
