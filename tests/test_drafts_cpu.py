"""What the operators of drafted tokens refuse, before any launch (CPU only)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from ab_attention import _lib, streaming
from ab_attention.streaming import (DraftTree, PagedCache, StreamingAttention, copy_pages, draft_tree, keep_drafts,
                                    tree_attention, verify_drafts)

BF16 = torch.bfloat16


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _i(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def _refuses(call, args, change, msg):
    args.update(change)
    with pytest.raises(ValueError, match=msg):
        call(**args)


@pytest.mark.parametrize("change,msg", [
    (dict(parents=_i(5, dtype=torch.int64)), "int32"), (dict(parents=_i(5, 1)), "one dim"), (dict(lengths=_i(4)[::2]), "contiguous"),
    (dict(offsets=_i(2)), "one batch"), (dict(offsets=_z(3, dtype=torch.float32)), "int32"), ({}, "CUDA")])
def test_draft_tree_refuses(change, msg):
    _refuses(draft_tree, dict(parents=_i(5), lengths=_i(2), offsets=_i(3)), change, msg)


def _tree(n):
    return DraftTree(_i(n), _i(n, dtype=torch.int64), _i(n))


@pytest.mark.parametrize("change,msg", [
    (dict(tree=_tree(4)), "Q's packed"), (dict(tree=DraftTree(_i(5), _i(5), _i(5))), "Q's packed"),
    (dict(tree=DraftTree(_i(5, dtype=torch.int64), _i(5, dtype=torch.int64), _i(5))), "int32"),
    (dict(tree=DraftTree(_i(5), _i(10, dtype=torch.int64)[::2], _i(5))), "Q's packed"), ({}, "CUDA")])
def test_tree_attention_refuses(change, msg):
    _refuses(tree_attention, dict(q=_z(5, 4, 64), cache=PagedCache(_z(3, 2, 8, 64), _z(3, 2, 8, 64)), page_table=_i(1, 2),
                                  lengths=_i(1), offsets=_i(2), tree=_tree(5)), change, msg)


@pytest.mark.parametrize("change,msg", [
    (dict(q=_z(5, 64)), "T,H,D"), (dict(q=_z(5, 3, 64)), "multiple"), (dict(window=0), "window"), (dict(frame=0), "frame"),
    (dict(q=_z(5, 4, 64, dtype=torch.float32)), "BF16"), (dict(sinks=-1), "sinks"), (dict(scale=float("nan")), "scale"),
    (dict(out=_z(5, 4, 128)), "out must"), (dict(out=_z(1, 4, 64).expand(5, 4, 64)), "out must"),
    (dict(out=_z(5, 4, 64).requires_grad_()), "requires a gradient")])
def test_tree_attention_refuses_as_chunk_attention(monkeypatch, change, msg):
    monkeypatch.setattr(streaming, "_gpu", lambda name, first, *others: first.device)
    monkeypatch.setattr(streaming, "_run", lambda *args: None)
    args = dict(q=_z(5, 4, 64), cache=PagedCache(_z(3, 2, 8, 64), _z(3, 2, 8, 64)), page_table=_i(1, 2), lengths=_i(1),
                offsets=_i(2), tree=_tree(5))
    assert tree_attention(**args).shape == (5, 4, 64)
    _refuses(tree_attention, args, change, msg)


_F = torch.float32


@pytest.mark.parametrize("change,msg", [
    (dict(target=_z(5, dtype=_F)), "T,V"), (dict(draft=_z(5, 8, dtype=_F)), "one shape"), (dict(draft=_z(5, 9)), "one type"),
    (dict(target=_z(5, 9, dtype=torch.float64), draft=None), "BF16"), (dict(target=_z(5, 0, dtype=_F), draft=None), "at least one token"),
    (dict(tokens=_i(5, dtype=torch.int16)), "int64"), (dict(uniforms=_z(5, dtype=torch.float64)), "float32"),
    (dict(tokens=_i(4)), "must be \\[5\\]"), (dict(parents=_i(6)), "must be \\[5\\]"), (dict(uniforms=_z(5, 1, dtype=_F)), "must be \\[5\\]"),
    (dict(parents=_i(5, dtype=torch.int64)), "int32"), (dict(offsets=_i(0)), "B\\+1"), ({}, "CUDA")])
def test_verify_drafts_refuses(change, msg):
    _refuses(verify_drafts, dict(target=_z(5, 9, dtype=_F), draft=_z(5, 9, dtype=_F), tokens=_i(5), parents=_i(5), offsets=_i(2),
                                 uniforms=_z(5, dtype=_F)), change, msg)


_CACHES = [
    ((_z(3, 2, 64), _z(3, 2, 64)), "layers,pages"), ((_z(3, 2, 8, 64), _z(3, 2, 16, 64)), "layers,pages"),
    ((_z(3, 2, 8, 96), _z(3, 2, 8, 96)), "64 or 128"), ((_z(3, 2, 8, 64), _z(3, 2, 8, 64, dtype=torch.float16)), "BF16"),
    ((_z(3, 2, 8, 64, dtype=_F), _z(3, 2, 8, 64, dtype=_F)), "BF16"), ((_z(3, 2, 12, 64), _z(3, 2, 12, 64)), "multiple of 8"),
    ((_z(3, 0, 8, 64), _z(3, 0, 8, 64)), "one head"), ((_z(3, 2, 8, 128)[..., ::2], _z(3, 2, 8, 64)), "rows must"),
    ((_z(3, 2, 8, 64), _z(8 * 3 * 2 * 64 + 4)[4:].reshape(3, 2, 8, 64)), "rows must"),
    ((_z(1, 2, 8, 64).expand(3, 2, 8, 64), _z(3, 2, 8, 64)), "overlap"), ((_z(2, 3, 2, 8, 64), _z(1, 3, 2, 8, 64).expand(2, 3, 2, 8, 64)), "overlap"),
    ((_z(3, 2, 8, 64), _z(3, 2, 8, 64)), "CUDA"), ((_z(2, 3, 2, 8, 64), _z(2, 3, 2, 8, 64)), "CUDA")]


@pytest.mark.parametrize("cache,msg", _CACHES)
def test_caches_that_are_refused(cache, msg):
    cache = PagedCache(*cache)
    with pytest.raises(ValueError, match=msg):
        copy_pages(cache, [(0, 1)])
    with pytest.raises(ValueError, match=msg):
        keep_drafts(cache, _i(1, 2), _i(1), _i(2), _i(5), _i(1))


@pytest.mark.parametrize("moves,msg", [([(0, 3)], "from 0 to 2"), ([(-1, 2)], "from 0 to 2"), ([(0, 1), (2, 1)], "only once"),
                                       ([(0, 1), (1, 2)], "only once"), ([(1, 1)], "only once"), ([(0, 1, 2)], "unpack"),
                                       ([(0,)], "unpack")])
def test_moves_that_are_refused(moves, msg):
    with pytest.raises(ValueError, match=msg):
        copy_pages(PagedCache(_z(3, 2, 8, 64), _z(3, 2, 8, 64)), moves)


@pytest.mark.parametrize("change,msg", [
    (dict(page_table=_i(2)), "page_table"), (dict(page_table=_i(1, 2, dtype=torch.int64)), "page_table"),
    (dict(page_table=_i(2, 2)), "one batch"), (dict(counts=_i(2)), "one batch"), (dict(offsets=_i(3)), "one batch"),
    (dict(path=_i(5, dtype=torch.int64)), "int32"), (dict(counts=_i(1, 1)), "one dim")])
def test_keep_drafts_refuses(change, msg):
    _refuses(keep_drafts, dict(cache=PagedCache(_z(3, 2, 8, 64), _z(3, 2, 8, 64)), page_table=_i(1, 2), lengths=_i(1), offsets=_i(2),
                               path=_i(5), counts=_i(1)), change, msg)


def test_what_autograd_is_told(monkeypatch):
    monkeypatch.setattr(streaming, "_gpu", lambda name, first, *others: first.device)
    monkeypatch.setattr(streaming, "_call", lambda *args: None)
    base = _z(2, 2, 3, 2, 8, 64)
    cache = PagedCache(base[:, 0], base[:, 1])
    calls = (lambda c: copy_pages(c, [(0, 1)]), lambda c: keep_drafts(c, _i(1, 2), _i(1), _i(2), _i(5), _i(1)))
    for call in calls:
        before = base._version
        assert call(cache) is cache and base._version > before
        with pytest.raises(ValueError, match="requires a gradient"):
            call(PagedCache(_z(3, 2, 8, 64), _z(3, 2, 8, 64).requires_grad_()))
        with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call(PagedCache(_z(3, 2, 8, 64), forward_ad.make_dual(_z(3, 2, 8, 64), _z(3, 2, 8, 64))))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        p = _z(5, 9, dtype=_F)
        verify_drafts(forward_ad.make_dual(p, p), None, _i(5), _i(5), _i(2), _z(5, dtype=_F))


# ---- the library's own checks ---------------------------------------------------

_A = 4096  # a 16-byte aligned stand-in address: every case is rejected before any runtime call


def _check(entry, kind, fields, change, msg):
    args = kind()
    for name, value in {**fields, **change}.items():
        where = args
        *outer, name = name.split(".")
        for part in outer:
            where = getattr(where, part)
        setattr(where, name, (ctypes.c_int64 * 3)(*value) if isinstance(value, tuple) else value)
    lib = _lib.load()
    assert getattr(lib, entry)(ctypes.byref(args), None) == 1
    assert msg in lib.ab_last_error(), lib.ab_last_error()


@pytest.mark.parametrize("change,msg", [(dict(batch=-1), b"too many"), (dict(batch=65536), b"too many"), (dict(tokens=1 << 30), b"too many"),
                                        (dict(parents=0), b"null"), (dict(above=0), b"null")])
def test_library_draft_tree(change, msg):
    fields = dict(parents=_A, lengths=_A, offsets=_A, positions=_A, near=_A, above=_A, batch=2, tokens=5)
    _check("ab_draft_tree", _lib.DraftTreeArgs, fields, change, msg)


@pytest.mark.parametrize("change,msg", [({"near": 0}, b"null"), ({"positions": 0}, b"null"), ({"chunk.dim": 96}, b"64 or 128"),
                                        ({"chunk.lengths": 0}, b"null"), ({"chunk.page_tokens": 12}, b"multiple of 8"),
                                        ({"chunk.workspace": 0}, b"null"), ({"chunk.workspace_bytes": 8}, b"smaller"),
                                        ({"chunk.workspace": _A + 8}, b"aligned")])
def test_library_tree_attention(change, msg):
    fields = {"positions": _A, "near": _A, "above": _A}
    chunk = dict(q=_A, k=_A, v=_A, out=_A, workspace=_A, workspace_bytes=1 << 30, lengths=_A, offsets=_A, page_table=_A, batch=1, heads=2, kv_heads=1, tokens=5, dim=64,
                 pages=3, page_tokens=8, table_width=2, frame=1, scale=0.1, q_stride=(0, 64, 128), k_stride=(512, 512, 64),
                 v_stride=(512, 512, 64), out_stride=(0, 64, 128))
    _check("ab_tree_attention", _lib.TreeArgs, {**{f"chunk.{k}": v for k, v in chunk.items()}, **fields}, change, msg)


@pytest.mark.parametrize("change,msg", [
    (dict(vocab=0), b"positive"), (dict(rows=-1), b"positive"), (dict(vocab=1 << 30), b"too many"), (dict(dtype=3), b"dtype"),
    (dict(target_stride=-1), b"strides"), (dict(draft_stride=1 << 40), b"strides"), (dict(target=0), b"null"), (dict(path=0), b"null"),
    (dict(workspace=0), b"null"), (dict(workspace_bytes=8), b"smaller"), (dict(workspace=_A + 8), b"misaligned"),
    (dict(target=_A + 2), b"misaligned"), (dict(draft=_A + 1, dtype=0), b"misaligned")])
def test_library_verify_drafts(change, msg):
    fields = dict(target=_A, draft=_A, tokens=_A, parents=_A, offsets=_A, uniforms=_A, path=_A, counts=_A, next=_A, batch=2, rows=5,
                  vocab=9, dtype=2, wide_tokens=1, target_stride=9, draft_stride=9, workspace=_A, workspace_bytes=1 << 20)
    _check("ab_verify_drafts", _lib.VerifyArgs, fields, change, msg)


_POOL = dict(k_cache=_A, v_cache=_A, layers=2, kv_heads=2, dim=64, pages=3, page_tokens=8, k_layer=4096, v_layer=4096,
             k_stride=(1024, 512, 64), v_stride=(1024, 512, 64))


@pytest.mark.parametrize("change,msg", [
    (dict(layers=0), b"layers"), (dict(layers=40000), b"layers"), (dict(k_layer=4), b"multiples of 8"), (dict(v_layer=-8), b"multiples of 8"),
    (dict(dim=32), b"64 or 128"), (dict(page_tokens=4), b"multiple of 8"), (dict(k_stride=(1024, 512, 60)), b"strides"),
    (dict(path=0), b"null"), (dict(k_cache=0), b"null"), (dict(v_cache=_A + 8), b"aligned"), (dict(lengths=0), b"null"),
    (dict(table_width=1 << 28), b"2^30")])
def test_library_keep_drafts(change, msg):
    fields = dict(_POOL, lengths=_A, offsets=_A, page_table=_A, path=_A, counts=_A, batch=1, tokens=5, table_width=2)
    _check("ab_keep_drafts", _lib.KeepArgs, fields, change, msg)


@pytest.mark.parametrize("change,msg", [
    (dict(layers=0), b"layers"), (dict(count=-1), b"page"), (dict(kv_heads=60000, page_tokens=1 << 20, k_stride=(0, 64, 64), v_stride=(0, 64, 64)), b"page"),
    (dict(moves=0), b"null"), (dict(k_cache=_A + 8), b"aligned"), (dict(pages=2), b"no page 2")])
def test_library_copy_pages(change, msg):
    moves = (ctypes.c_int32 * 4)(0, 1, 0, 2)
    _check("ab_copy_pages", _lib.CopyArgs, dict(_POOL, moves=ctypes.addressof(moves), count=2), change, msg)


# ---- StreamingAttention ---------------------------------------------------------


def test_steps_of_drafts_refuse():
    stream = StreamingAttention(1, 3, 1, 4, 16, dim=64, device="cpu")
    before = (list(stream.free), list(stream.tokens), [dict(h) for h in stream.held])
    for new, parents, msg in (([2, 0, 1], [[-1, 0], []], "parents must give"), ([2, 0, 1], [[-1, 0], [], [-1, 0]], "parents must give"),
                              ([2, 0, 1], [[-1, 1], [], [-1]], "come before"), ([1, 0, 1], [[-2], [], [-1]], "come before")):
        with pytest.raises(ValueError, match=msg):
            stream.begin(new, parents)
    with pytest.raises(ValueError, match="after begin"):
        stream.keep(_i(3), _i(3))
    stream.offsets, stream.step_tokens, stream.tree = _i(4), 3, _tree(3)
    with pytest.raises(ValueError, match="counts"):
        stream.keep(_i(3), _i(2))
    with pytest.raises(ValueError, match="path"):
        stream.keep(_i(2), _i(3))
    stream.new = [2, 0, 1]
    with pytest.raises(ValueError, match="counts must be"):
        stream.keep(_i(3), torch.tensor([1, 0, 2]))
    for call in (lambda: stream.begin([1, 1, 1]), lambda: stream.fork(0, 1)):
        with pytest.raises(ValueError, match="keep comes before"):
            call()
    assert before == (stream.free, stream.tokens, stream.held)


def test_forks_share_pages():
    stream = StreamingAttention(1, 3, 1, 4, 16, dim=64, device="cpu")
    stream.held[0], stream.tokens[0], stream.free = {0: 3, 1: 2}, 20, [1, 0]
    stream.owners = [0, 0, 1, 1]
    stream.fork(0, 2)
    assert stream.held[2] == {0: 3, 1: 2} and stream.tokens == [20, 0, 20] and stream.owners == [0, 0, 2, 2]
    with pytest.raises(ValueError, match="without tokens"):
        stream.fork(0, 2)
    with pytest.raises(ValueError, match="without tokens"):
        stream.fork(0, 0)
    stream.finish(0)
    assert stream.free == [1, 0] and stream.owners == [0, 0, 1, 1] and stream.tokens == [0, 0, 20]
    stream.finish(2)
    assert sorted(stream.free) == [0, 1, 2, 3]
