"""Attention of video that is made (or trained) frame by frame: rotary positions
over (time, height, width), attention that is causal over frames with a sliding
window and first frames that stay visible, and the same attention of new tokens
over a paged cache.

The mask of all of them: tokens are grouped into frames of ``frame`` tokens
(``frame=1``: plain causal attention), and the query at position p sees the key
at position t where

    t // frame <= p // frame  and
    (p // frame - t // frame < window  or  t // frame < sinks)

so ``window`` and ``sinks`` count frames; ``window=None`` is no limit. A query
that sees nothing gets o = 0 and lse = -inf.

Serving: ``rotary`` of the new tokens' Q and K, ``append_cache``, then
``chunk_attention``, or ``StreamingAttention``, which makes the three calls and
keeps the page table. Training: ``rotary`` and ``window_attention``. The
reference has no counterpart: its attention sees a whole clip at once.

A step that checks several drafted tokens at once: ``draft_tree`` (for ``rotary`` the
positions), in every layer ``append_cache`` and ``tree_attention``, then
``verify_drafts`` on the model's probabilities and ``keep_drafts``. ``copy_pages`` is
for sequences that are continued in several ways from a common beginning.

Everything runs on the current stream of the tensors' device and synchronises
nothing; sizes that are on the device (lengths, offsets, page tables) are
bounded by the kernels and never read on the host.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_MOST = 1 << 30
_REACH = (1 << 31) - 128  # 16-bit elements


def _strided(t: torch.Tensor, align: int = 8) -> torch.Tensor:
    """t itself where its rows (last dim contiguous, starting on 16 bytes) can be
    read where they lie, else a contiguous copy; of [B, H, N, D] the kernels reach
    4 GiB from a head's first row on."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        strides = t.stride()
        if strides[-1] == 1 and not any(n > 1 and s % align for n, s in zip(t.shape, strides[:-1])) and (
                strides[-2] * (t.shape[-2] + 64) < _REACH or t.ndim == 3):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _gpu(name: str, first, *others):
    device = first.device
    if device.type != "cuda":
        raise ValueError(f"{name} requires tensors on one CUDA device")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{name} requires tensors on one CUDA device")
    return device


def _no_tangent(name: str, *tensors):
    """Refuses tensors with a forward-mode tangent, which the kernels would drop."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise ValueError(f"{name} has no forward-mode derivative")


def _own_rows(t: torch.Tensor) -> bool:
    """Whether no two rows of t (its last dim contiguous) share memory: from the smallest
    stride up, each reaches past all that the smaller ones span."""
    if t.is_contiguous():
        return True
    span = t.shape[-1]
    for stride, n in sorted((s, n) for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        if stride < span:
            return False
        span += stride * (n - 1)
    return True


def _writes(name: str, *tensors):
    """Tells autograd of writes that go past it, as torch's in-place operations do, so
    that a gradient which still needs the old values raises."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} cannot write to a tensor that requires a gradient")
    increment_version([t for t in tensors if not t.is_inference()])


def _bytes_at(data: bytes) -> int:
    """The address of the bytes, which live as long as ``data``."""
    return ctypes.cast(data, ctypes.c_void_p).value


def _call(entry: str, device, packed: bytes):
    with _lib.on(device):
        status = _lib.raw(entry)(packed, _lib.raw_stream(device))
    if status:
        _lib.check(status)


_ROTARY, _WINDOW, _APPEND = map(_lib.packer, (_lib.RotaryArgs, _lib.WindowArgs, _lib.AppendArgs))
_TREE, _VERIFY, _KEEP, _COPY = map(_lib.packer, (_lib.DraftTreeArgs, _lib.VerifyArgs, _lib.KeepArgs, _lib.CopyArgs))
_TREE_REST = struct.Struct("=3Q")     # ab_tree_args behind its chunk
_GRAD_REST = struct.Struct("=5Q12q")  # ab_window_grad_args behind its forward part
_WORKSPACE = struct.Struct("=2Q")     # the last fields of ab_window_args and ab_verify_args
_ZERO = (0, 0, 0)


# ---- rotary positions ---------------------------------------------------------


def _rotate(q, k, positions, axes, theta, halves, joint, inverse):
    align = 4 if q.dtype == torch.float32 else 8
    q = _strided(q, align)
    q_out = torch.empty_like(q)
    batch, heads, tokens, dim = q.shape
    k_out, k_at, k_out_at, k_heads, k_stride, k_out_stride = None, 0, 0, 0, _ZERO, _ZERO
    if k is not None:
        k = _strided(k, align)
        k_out = torch.empty_like(k)
        k_at, k_out_at, k_heads, k_stride, k_out_stride = (k.data_ptr(), k_out.data_ptr(), k.shape[1], k.stride()[:3],
                                                           k_out.stride()[:3])
    _call("ab_rotary", q.device, _ROTARY.pack(
        q.data_ptr(), k_at, q_out.data_ptr(), k_out_at, positions.data_ptr(), batch, heads, k_heads, tokens, dim,
        _DTYPES[q.dtype], *q.stride()[:3], *k_stride, *q_out.stride()[:3], *k_out_stride, len(axes), *axes,
        *(0,) * (4 - len(axes)), theta, joint, halves, _POSITIONS[positions.dtype], positions.ndim == 3, inverse))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, *how):
        ctx.save_for_backward(positions)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, *how, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        _no_tangent("the gradient of rotary", dq, dk)
        (positions,) = ctx.saved_tensors
        if dq is None:  # only K's result was used
            dq, dk = dk, None
            flipped = True
        else:
            flipped = False
        grads = (None, None) if dq is None else _rotate(dq, dk, positions, *ctx.how, True)
        if flipped:
            grads = grads[::-1]
        return (*grads, *[None] * (len(ctx.how) + 1))


@functools.lru_cache(maxsize=64)
def _axes(axes, dim, pairing):
    """axes, checked."""
    if not 1 <= len(axes) <= 4 or any(a <= 0 or a % 2 for a in axes) or sum(axes) > dim:
        raise ValueError("axes must be 1 to 4 positive even numbers of dims that add up to at most D")
    if pairing not in ("adjacent", "halves"):
        raise ValueError("pairing must be 'adjacent' or 'halves'")
    if pairing == "halves" and sum(axes) % 16:
        raise ValueError("pairing 'halves' requires a multiple of 16 turned dims")
    return axes


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes, *, theta: float = 10000.0,
           pairing: str = "adjacent", joint: bool = False):
    """q [B, H, N, D] and k [B, Hk, N, D] (or None) with rotary positions over several axes.

    ``positions`` [N, A] or [B, N, A] (int32, int64 or float32) gives every token's
    place on A <= 4 axes, for example (time, height, width); ``axes`` gives the
    dims that each axis turns, even numbers that add up to at most D (Wan2.1:
    (44, 42, 42), HunyuanVideo: (16, 56, 56)). The j-th pair of an axis of d dims
    turns by position * theta^(-2j/d); with ``joint`` the i-th pair of all axes by
    position * theta^(-2i/sum(axes)). ``pairing`` "adjacent" pairs values 2i and
    2i + 1, "halves" values i and i + sum(axes)/2 (a sum divisible by 16). Dims
    behind the axes' stay as they are. D is a multiple of 8; bf16, fp16 or float32.

    Returns (q, k) as new tensors (k None if it was), in the memory order of the
    inputs. Differentiable in q and k (the gradient is the opposite rotation), in
    reverse mode only.
    """
    if q.ndim != 4 or (k is not None and (k.ndim != 4 or k.shape[::2] != q.shape[::2] or k.shape[3] != q.shape[3])):
        raise ValueError("rotary requires Q [B,H,N,D] and K [B,Hk,N,D] of the same batch, tokens and dim")
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
        raise ValueError("rotary requires BF16, FP16 or FP32 Q/K of one type")
    batch, _, tokens, dim = q.shape
    if dim % 8 or dim > 1024:
        raise ValueError("rotary requires a head dim that is a multiple of 8, at most 1024")
    axes = _axes(tuple(map(int, axes)), dim, pairing)
    theta = float(theta)
    if not math.isfinite(theta) or theta <= 0:
        raise ValueError("theta must be positive and finite")
    if positions.dtype not in _POSITIONS:
        raise ValueError("positions must be int32, int64 or float32")
    shape = positions.shape
    if shape != (tokens, len(axes)) and shape != (batch, tokens, len(axes)):
        raise ValueError(f"positions must be [{tokens}, {len(axes)}] or [{batch}, {tokens}, {len(axes)}]")
    _no_tangent("rotary", q, k, positions)
    _gpu("rotary", q, k, positions)
    if q.shape[1] == 0 or (k is not None and k.shape[1] == 0):
        raise ValueError("rotary requires at least one head")
    how = (axes, theta, pairing == "halves", bool(joint))
    positions = positions.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, *how)
    return _rotate(q, k, positions, *how, False)


# ---- windowed attention -------------------------------------------------------


def _mask(window, sinks, frame):
    """(window, 0 for no limit, sinks, frame) as checked numbers."""
    window = 0 if window is None else min(int(window), _MOST)
    sinks, frame = int(sinks), int(frame)
    if frame < 1:
        raise ValueError("frame must be at least one token")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    return window, min(sinks, _MOST), min(frame, _MOST)


def _check_window(window, scale, dim):
    if window is not None and int(window) < 1:
        raise ValueError("window must be at least one frame, or None")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return scale


def _run(entry, device, packed, behind=b"", asks="ab_window_workspace_bytes"):
    """One call with the workspace that it ``asks`` for, the last two fields of ``packed``, which lives for the call
    only; ``behind``: fields after those."""
    with _lib.on(device):
        size = _lib.raw(asks)(packed + behind)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            packed = packed[:-_WORKSPACE.size] + _WORKSPACE.pack(workspace.data_ptr(), size)
        status = _lib.raw(entry)(packed + behind, _lib.raw_stream(device))
    if status:
        _lib.check(status)


def _window_args(q, k, v, out, rest, lse, lengths, window, sinks, frame, scale, workspace=0, size=0):
    """The call's ab_window_args of [B, H, N, D] tensors that _strided has seen."""
    batch, heads, tokens, dim = q.shape
    return _WINDOW.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if rest is None else rest.data_ptr(),
                        0 if lse is None else lse.data_ptr(), 0 if lengths is None else lengths.data_ptr(), 0, 0, batch, heads, k.shape[1], tokens, dim,
                        _DTYPES[q.dtype], 0, 0, 0, window, sinks, frame, scale, *q.stride()[:3], *k.stride()[:3],
                        *v.stride()[:3], *out.stride()[:3], workspace, size)


def _window_forward(q, k, v, lengths, window, sinks, frame, scale, return_lse, rest=None):
    out = torch.empty_like(q)
    lse = q.new_empty(q.shape[:3], dtype=torch.float32) if return_lse else None
    if out.numel():
        _run("ab_window_attention", q.device, _window_args(q, k, v, out, rest, lse, lengths, window, sinks, frame, scale))
    return out, lse


class _Window(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, *how):
        q, k, v = _strided(q), _strided(k), _strided(v)
        rest = torch.empty_like(q)  # what out's rounding takes: delta is made of both
        out, lse = _window_forward(q, k, v, lengths, *how, True, rest)
        ctx.save_for_backward(q, k, v, out, rest, lse, lengths)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        _no_tangent("the gradient of window attention", dout, dlse)
        q, k, v, out, rest, lse, lengths = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * (4 + len(ctx.how))
        dout = torch.zeros_like(out) if dout is None else _strided(dout)
        dlse = None if dlse is None else dlse.contiguous()
        grads = tuple(torch.empty_like(t) for t in (q, k, v))
        if q.numel():
            behind = _GRAD_REST.pack(dout.data_ptr(), 0 if dlse is None else dlse.data_ptr(), *(g.data_ptr() for g in grads),
                                     *dout.stride()[:3], *(s for g in grads for s in g.stride()[:3]))
            tensors = (q, k, v, out, rest, lse, lengths, *ctx.how)
            size = _lib.raw("ab_window_grad_workspace_bytes")(_window_args(*tensors) + behind)
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            _call("ab_window_attention_grad", q.device, _window_args(*tensors, workspace.data_ptr(), size) + behind)
        return (*grads, *[None] * (1 + len(ctx.how)))


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     frame: int = 1, lengths: torch.Tensor | None = None, scale: float | None = None,
                     return_lse: bool = False):
    """Attention of q [B, H, N, D] over k, v [B, Hk, N, D] that is causal over
    frames with a sliding window and sinks (the mask above; token t is at position
    t). D is 64 or 128, bf16 or fp16; H is a multiple of Hk, and query head h reads
    key head h // (H // Hk). ``lengths`` int32 [B] are the batch items' tokens: the
    ones behind them are padding that nothing reads, with o = 0 and lse = -inf.
    ``scale`` defaults to D ** -0.5.

    Returns o in q's type and memory order, and with ``return_lse`` the base-2
    softmax normaliser as float32 [B, H, N]. Differentiable in q, k and v, through
    both, in reverse mode only; the same inputs give the same gradients bit for bit. In fp16 the logits'
    gradients are rounded to fp16 on their way, so the losses of small gradients
    want the scaling that is usual in fp16. Values that are not
    finite reach the results of the queries that see them only, but may reach any
    gradient of their batch item.
    """
    if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape:
        raise ValueError("Q [B,H,N,D] and K/V [B,Hk,N,D] must share batch, tokens and dim")
    batch, heads, tokens, dim = q.shape
    kv_heads = k.shape[1]
    if k.shape != (batch, kv_heads, tokens, dim):
        raise ValueError("Q [B,H,N,D] and K/V [B,Hk,N,D] must share batch, tokens and dim")
    if dim != 128 and dim != 64:
        raise ValueError("window attention requires head_dim 64 or 128")
    dtype = q.dtype
    if (dtype != torch.bfloat16 and dtype != torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("window attention requires BF16 or FP16 Q/K/V of one type")
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("the query heads must be a positive multiple of the key heads")
    scale = _check_window(window, scale, dim)
    window, sinks, frame = _mask(window, sinks, frame)
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != q.shape[:1] or not lengths.is_contiguous()):
        raise ValueError("lengths must be int32 [B]")
    _no_tangent("window attention", q, k, v)
    _gpu("window attention", q, k, v, lengths)
    how = (window, sinks, frame, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Window.apply(q, k, v, lengths, *how)
    else:
        out, lse = _window_forward(_strided(q), _strided(k), _strided(v), lengths, *how, return_lse)
    return (out, lse) if return_lse else out


# ---- paged cache --------------------------------------------------------------


class PagedCache(NamedTuple):
    """Keys and values of many sequences in pages: two tensors [pages, heads, page
    tokens, D] (or views of that shape of any memory order with rows of D), page
    tokens a multiple of 8. Which page holds which tokens of which sequence is the
    page table's: int32 [sequences, width], entry (b, i) the page of the positions
    i * page tokens .. + page tokens - 1, or any number outside [0, pages) for
    none, as of pages that have been given back."""

    k: torch.Tensor
    v: torch.Tensor


def _check_cache(name, x, cache, page_table, lengths, offsets):
    """The checks of packed tokens x and what belongs to a cache; the cache's heads."""
    if x.ndim != 3:
        raise ValueError(f"{name} requires packed tokens [T,H,D]")
    heads, dim = x.shape[1], x.shape[2]
    k, v = cache
    if k.ndim != 4 or k.shape != v.shape or k.shape[3] != dim:
        raise ValueError("the cache must be two [pages,heads,page tokens,D] tensors with the tokens' D")
    if dim != 128 and dim != 64:
        raise ValueError(f"{name} requires head_dim 64 or 128")
    dtype = x.dtype
    if (dtype != torch.bfloat16 and dtype != torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{name} requires BF16 or FP16 tokens and a cache of the same type")
    _, kv_heads, page, _ = k.shape
    if page == 0 or page % 8:
        raise ValueError("pages must hold a positive multiple of 8 tokens")
    for t in cache:
        if t.data_ptr() % 16 or not (t.is_contiguous() or (
                t.stride(3) == 1 and not any(n > 1 and s % 8 for n, s in zip(t.shape, t.stride()[:3])))):
            raise ValueError("the cache's rows must be contiguous and start on 16 bytes")
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("the query heads must be a positive multiple of the cache's heads")
    if page_table.ndim != 2 or lengths.ndim != 1 or offsets.ndim != 1 or not (
            page_table.shape[0] == lengths.shape[0] == offsets.shape[0] - 1):
        raise ValueError("page_table [B,width], lengths [B] and offsets [B+1] must be of one batch")
    for t in (page_table, lengths, offsets):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("page_table, lengths and offsets must be contiguous int32")
    _no_tangent(name, x, k, v)
    _gpu(name, x, k, v, page_table, lengths, offsets)
    return kv_heads


def append_cache(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 offsets: torch.Tensor) -> PagedCache:
    """Writes the new keys and values k, v [T, heads, D] into the cache, in place.

    Sequence b's new tokens are the rows offsets[b] .. offsets[b + 1] - 1 (int32
    [B + 1], ascending, bounded to 0 .. T); ``lengths`` int32 [B] are the tokens of
    each sequence with the new ones, so that its last row goes to position
    lengths[b] - 1. Rows whose entry in the page table is no page are dropped.
    Returns the cache; k and v share no memory with it. Not differentiable: no
    gradient reaches k and v by it.
    """
    if k.shape != v.shape or v.dtype != k.dtype:
        raise ValueError("K and V must be packed tokens [T,H,D] of one shape and type")
    if _check_cache("append_cache", k, cache, page_table, lengths, offsets) != k.shape[1]:
        raise ValueError("K and V must have the cache's heads")
    if not (_own_rows(cache.k) and _own_rows(cache.v)):
        raise ValueError("append_cache cannot write to an expanded cache or one whose rows overlap")
    _no_tangent("append_cache", v)
    device = k.device
    if v.device != device:
        raise ValueError("append_cache requires tensors on one CUDA device")
    k, v = _strided(k), _strided(v)
    _writes("append_cache", *cache)
    pages, heads, page, dim = cache.k.shape
    _call("ab_append_cache", device, _APPEND.pack(
        k.data_ptr(), v.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), lengths.data_ptr(), offsets.data_ptr(),
        page_table.data_ptr(), page_table.shape[0], heads, k.shape[0], dim, pages, page, page_table.shape[1],
        0, k.stride(1), k.stride(0), 0, v.stride(1), v.stride(0), *cache.k.stride()[:3], *cache.v.stride()[:3]))
    return cache


def chunk_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                    offsets: torch.Tensor, *, window: int | None = None, sinks: int = 0, frame: int = 1,
                    scale: float | None = None, return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of the sequences' new tokens q [T, H, D] over their cached keys
    and values, the new ones among them (``append_cache`` first; ``lengths`` and
    ``offsets`` as there). A sequence may bring one token or a whole prompt; query i
    of n is at position lengths[b] - n + i of the mask above. Keys in places that
    the page table gives no page are not seen, and nothing outside of the pages'
    visible tokens is read. D is 64 or 128, bf16 or fp16; H is a multiple of the
    cache's heads. Not differentiable: the result never requires a gradient, also
    where q or the cache does (train with ``window_attention``).

    Returns o [T, H, D] and with ``return_lse`` the base-2 normaliser float32
    [T, H]. Rows outside of offsets[0] .. offsets[B] - 1 are not written (with
    ``out``, a tensor of q's shape and type to write to, they stay as they are).
    ``out`` may be q itself; it shares no memory with anything else that is read.
    """
    return _over_cache("chunk attention", ("ab_chunk_attention",), q, cache, page_table, lengths, offsets, window, sinks, frame,
                       scale, return_lse, out)


def _over_cache(name, entry, q, cache, page_table, lengths, offsets, window, sinks, frame, scale, return_lse, out, *behind):
    """``entry``: the library's, and the one that says its workspace's size if it is another; ``behind``: bytes of its
    arguments after ab_window_args."""
    _check_cache(name, q, cache, page_table, lengths, offsets)
    device = q.device
    scale = _check_window(window, scale, q.shape[-1])
    window, sinks, frame = _mask(window, sinks, frame)
    q = _strided(q)
    tokens, heads, dim = q.shape
    if out is None:
        out = q.new_empty((tokens, heads, dim))
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != device or out.data_ptr() % 8 or out.stride(2) != 1
          or any(n > 1 and s % 4 for n, s in zip(out.shape[:2], out.stride())) or not _own_rows(out)):
        raise ValueError("out must be of Q's shape, type and device, with contiguous rows that start on 8 bytes, each its own")
    else:
        _writes(name, out)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    if tokens and page_table.shape[0]:
        pages, kv_heads, page, _ = cache[0].shape
        k, v = cache
        _run(entry[0], device, _WINDOW.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, 0 if lse is None else lse.data_ptr(),
            lengths.data_ptr(), offsets.data_ptr(), page_table.data_ptr(), page_table.shape[0], heads, kv_heads, tokens, dim,
            _DTYPES[q.dtype], pages, page, page_table.shape[1], window, sinks, frame, scale, 0, q.stride(1), q.stride(0),
            *k.stride()[:3], *v.stride()[:3], 0, out.stride(1), out.stride(0), 0, 0), *behind, *entry[1:])
    return (out, lse) if return_lse else out


# ---- drafted tokens -----------------------------------------------------------


def _ints(name, **tensors):
    for what, t in tensors.items():
        if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous():
            raise ValueError(f"{name} requires {what} as a contiguous int32 tensor of one dim")


class DraftTree(NamedTuple):
    """``draft_tree``'s results, int32, int64 and int32 [T]. ``positions`` are the new
    tokens'. Which tokens are on the line down to each, itself too, is said by the places
    of ``near``'s bits (bit j: 64 (i // 64) + j for the token at place i) and by
    ``above``, the last place of the line before those 64, or -1."""

    positions: torch.Tensor
    near: torch.Tensor
    above: torch.Tensor


def draft_tree(parents: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor) -> DraftTree:
    """The tree that the sequences' new tokens are, for all layers of a step.

    Sequence b's n new tokens are the rows offsets[b] .. offsets[b + 1] - 1 (int32
    [B + 1]), of lengths[b] (int32 [B]) in all. ``parents`` int32 [T] gives for each
    the place, 0 .. n - 1, of the new token that it follows, which comes before it; any
    other number is none: the token follows the cached ones. A token with d others
    above it is at position lengths[b] - n + d, though its keys and values are in the
    cache's place lengths[b] - n + i, as ``append_cache`` puts them. Rows of no
    sequence get position 0.
    """
    _ints("draft_tree", parents=parents, lengths=lengths, offsets=offsets)
    if lengths.shape[0] != offsets.shape[0] - 1:
        raise ValueError("lengths [B] and offsets [B+1] must be of one batch")
    device = _gpu("draft_tree", parents, lengths, offsets)
    tokens, batch = parents.shape[0], lengths.shape[0]
    if batch == 0:
        return DraftTree(torch.zeros_like(parents), parents.new_zeros(tokens, dtype=torch.int64), torch.full_like(parents, -1))
    tree = DraftTree(torch.empty_like(parents), parents.new_empty(tokens, dtype=torch.int64), torch.empty_like(parents))
    if tokens:
        _call("ab_draft_tree", device, _TREE.pack(parents.data_ptr(), lengths.data_ptr(), offsets.data_ptr(),
                                                  *(t.data_ptr() for t in tree), batch, tokens))
    return tree


def tree_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                   offsets: torch.Tensor, tree: DraftTree, *, window: int | None = None, sinks: int = 0, frame: int = 1,
                   scale: float | None = None, return_lse: bool = False, out: torch.Tensor | None = None):
    """``chunk_attention`` of new tokens that are a tree (``draft_tree`` of the same
    ``lengths`` and ``offsets``; other values in it give other results, but reach no
    other memory): every token sees the cached ones that the mask gives its position,
    and of the new ones those above it and itself, as far as the mask gives it their
    positions. With ``frame`` above 1 a token sees no later ones of its frame, as
    those are drafts.
    """
    positions, near, above = tree
    _ints("tree attention", positions=positions, above=above)
    if near.dtype != torch.int64 or not near.is_contiguous() or not positions.shape == near.shape == above.shape == q.shape[:1]:
        raise ValueError("tree attention requires the tree of Q's packed tokens")
    _gpu("tree attention", q, *tree)
    return _over_cache("tree attention", ("ab_tree_attention", "ab_tree_workspace_bytes"), q, cache, page_table, lengths, offsets,
                       window, sinks, frame, scale, return_lse, out,
                       _TREE_REST.pack(positions.data_ptr(), near.data_ptr(), above.data_ptr()))


class Kept(NamedTuple):
    """``verify_drafts``' results: ``path`` int32 [T], from offsets[b] on the places of
    sequence b's kept tokens, then -1; ``counts`` int32 [B], how many; ``next`` [B], the
    token behind them, of the drafts' type."""

    path: torch.Tensor
    counts: torch.Tensor
    next: torch.Tensor


def verify_drafts(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, parents: torch.Tensor,
                  offsets: torch.Tensor, uniforms: torch.Tensor) -> Kept:
    """Which drafted tokens stay, and the token behind them, so that what is written is
    distributed as the target's probabilities say.

    The new tokens ``tokens`` [T] (int32 or int64), ``parents`` and ``offsets`` are as in
    ``draft_tree``; the first of each sequence is the one that was written last and is
    kept, the others hang below it. ``target`` [T, V] are the probabilities of what comes
    behind each (bf16, fp16 or float32; the values are taken as they are, rows need not
    add up to one exactly), ``draft`` of the same shape and type the ones that its
    children were drawn from, or None for children that were chosen without chance, such
    as the likeliest ones. ``uniforms`` float32 [T] are random numbers in [0, 1).

    From the last kept token on its children j are looked at in the order of their
    places. With w = target's row and S = 1 at first, j is kept where
    uniforms[j] * draft[tokens[j]] * S < w[tokens[j]] (None: draft = 1), and the walk goes
    on from it. Else w becomes max(w - S * draft, 0) and S its sum (where that is 0
    both stay as they are), or, chosen, S loses w[tokens[j]], which becomes 0. Where no
    child is left the next token is the first with w > 0 whose running sum of w passes
    uniforms[offsets[b]] times the whole sum (-1 where all w are 0). Sums are in 64
    bits. Values that are not positive and finite count as 0, tokens outside of
    0 .. V - 1 are never kept. A sequence without new tokens has counts 0 and next -1.
    """
    if target.ndim != 2 or (draft is not None and draft.shape != target.shape):
        raise ValueError("target and draft must be [T,V] probabilities of one shape")
    if target.dtype not in _DTYPES or (draft is not None and draft.dtype != target.dtype):
        raise ValueError("verify_drafts requires BF16, FP16 or FP32 probabilities of one type")
    rows, vocab = target.shape
    if vocab == 0:
        raise ValueError("verify_drafts requires at least one token in the vocabulary")
    _ints("verify_drafts", parents=parents, offsets=offsets)
    if tokens.dtype not in (torch.int32, torch.int64) or uniforms.dtype != torch.float32:
        raise ValueError("tokens must be int32 or int64, uniforms float32")
    if not tokens.shape == parents.shape == uniforms.shape == target.shape[:1]:
        raise ValueError(f"tokens, parents and uniforms must be [{rows}], as target has rows")
    if offsets.shape[0] == 0:
        raise ValueError("offsets must be [B+1]")
    _no_tangent("verify_drafts", target, draft, uniforms)
    device = _gpu("verify_drafts", target, draft, tokens, parents, offsets, uniforms)
    tokens, uniforms = tokens.contiguous(), uniforms.contiguous()
    target, draft = (t if t is None or t.stride(1) == 1 or vocab == 1 else t.contiguous() for t in (target, draft))
    batch = offsets.shape[0] - 1
    kept = Kept(torch.empty_like(parents), parents.new_empty(batch), tokens.new_empty(batch))
    if batch == 0:
        kept.path.fill_(-1)
        return kept
    path, counts, after = kept
    _run("ab_verify_drafts", device, _VERIFY.pack(
        target.data_ptr(), 0 if draft is None else draft.data_ptr(), tokens.data_ptr(), parents.data_ptr(), offsets.data_ptr(),
        uniforms.data_ptr(), path.data_ptr(), counts.data_ptr(), after.data_ptr(), batch, rows, vocab, _DTYPES[target.dtype],
        tokens.dtype == torch.int64, target.stride(0), 0 if draft is None else draft.stride(0), 0, 0), b"",
        "ab_verify_workspace_bytes")
    return kept


def _check_layers(name, cache):
    """(layers, sizes of a layer, strides of a layer in k and v, strides in a layer) of a cache of one layer, or of
    several, [layers, ..]."""
    k, v = cache
    shape, dtype = k.shape, k.dtype
    if not 4 <= len(shape) <= 5 or shape != v.shape:
        raise ValueError("the cache must be two [pages,heads,page tokens,D] or [layers,pages,heads,page tokens,D] tensors")
    pages, heads, page, dim = shape[-4:]
    if dim != 128 and dim != 64:
        raise ValueError(f"{name} requires head_dim 64 or 128")
    if (dtype != torch.bfloat16 and dtype != torch.float16) or v.dtype != dtype:
        raise ValueError(f"{name} requires a BF16 or FP16 cache")
    if page == 0 or page % 8:
        raise ValueError("pages must hold a positive multiple of 8 tokens")
    if heads == 0:
        raise ValueError("the cache must have at least one head")
    for t in cache:
        whole = t.is_contiguous()
        if t.data_ptr() % 16 or not (whole or (
                t.stride(-1) == 1 and not any(n > 1 and s % 8 for n, s in zip(shape, t.stride()[:-1])))):
            raise ValueError("the cache's rows must be contiguous and start on 16 bytes")
        if not (whole or _own_rows(t)):
            raise ValueError(f"{name} cannot write to an expanded cache or one whose rows overlap")
    if len(shape) == 4:
        return 1, (pages, heads, page, dim), (0, 0), k.stride()[:3], v.stride()[:3]
    a, b = k.stride(), v.stride()
    return shape[0], (pages, heads, page, dim), (a[0], b[0]), a[1:4], b[1:4]


def keep_drafts(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor,
                path: torch.Tensor, counts: torch.Tensor) -> PagedCache:
    """Moves the kept tokens' keys and values next to each other, in place.

    ``path`` int32 [T] and ``counts`` int32 [B] are ``verify_drafts``', the others those
    that the drafts were appended by: in sequence b, with n new tokens, the cache's
    position lengths[b] - n + path[offsets[b] + j] is copied to lengths[b] - n + j, for
    j < counts[b], so that the sequence goes on with lengths[b] - n + counts[b] tokens.
    Places outside of j .. n - 1 and ones on no page move nothing. The cache may be that of one
    layer or, as tensors [layers, pages, heads, page tokens, D], of all layers, which one
    call then takes. Its keys and values share no memory, and no page that has new tokens
    is in two places of the table. Returns the cache.
    """
    layers, (pages, heads, page, dim), layer_strides, k_stride, v_stride = _check_layers("keep_drafts", cache)
    if page_table.ndim != 2 or page_table.dtype != torch.int32 or not page_table.is_contiguous():
        raise ValueError("page_table must be contiguous int32 [B,width]")
    _ints("keep_drafts", lengths=lengths, offsets=offsets, path=path, counts=counts)
    batch = lengths.shape[0]
    if not page_table.shape[0] == offsets.shape[0] - 1 == counts.shape[0] == batch:
        raise ValueError("page_table [B,width], lengths [B], offsets [B+1] and counts [B] must be of one batch")
    k, v = cache
    if k.data_ptr() == v.data_ptr() and k.numel():
        raise ValueError("keep_drafts requires keys and values that share no memory")
    _no_tangent("keep_drafts", k, v)
    device = _gpu("keep_drafts", k, v, page_table, lengths, offsets, path, counts)
    _writes("keep_drafts", k, v)
    if layers:
        _call("ab_keep_drafts", device, _KEEP.pack(
            k.data_ptr(), v.data_ptr(), lengths.data_ptr(), offsets.data_ptr(), page_table.data_ptr(), path.data_ptr(),
            counts.data_ptr(), layers, batch, heads, path.shape[0], dim, pages, page, page_table.shape[1], *layer_strides,
            *k_stride, *v_stride))
    return cache


def copy_pages(cache: PagedCache, moves) -> PagedCache:
    """Copies pages to pages, in place: ``moves`` are pairs (from, to) of page numbers, on
    the host. A page that is copied to is named only once. The cache may be that of one
    layer or of all, as in ``keep_drafts``. Returns the cache. A call captured into a
    graph repeats the moves that it was captured with.
    """
    layers, (pages, heads, page, dim), layer_strides, k_stride, v_stride = _check_layers("copy_pages", cache)
    k, v = cache
    flat = [int(p) for source, target in moves for p in (source, target)]
    if flat and not (0 <= min(flat) and max(flat) < pages):
        raise ValueError(f"moves must name pages from 0 to {pages - 1}")
    to = set(flat[1::2])
    if 2 * len(to) != len(flat) or not to.isdisjoint(flat[::2]):
        raise ValueError("a page that is copied to must be named only once")
    _no_tangent("copy_pages", k, v)
    device = _gpu("copy_pages", k, v)
    _writes("copy_pages", k, v)
    if flat and layers:
        host = struct.pack(f"={len(flat)}i", *flat)  # read by the call itself
        _call("ab_copy_pages", device, _COPY.pack(
            k.data_ptr(), v.data_ptr(), _bytes_at(host), len(to), layers, heads, dim, pages, page, *layer_strides,
            *k_stride, *v_stride))
    return cache


class StreamingAttention:
    """The attention layers of a transformer that makes several videos (or texts)
    chunk by chunk: their paged caches, and one page table for all of them.

    A step is ``begin(new)``, with the new tokens of every sequence (0 for one that
    pauses), then in every layer ``attend(layer, q, k, v, positions)``. Pages are
    given out on the host as sequences grow, given back when no later query can see
    any of their tokens (behind the window, not among the sinks), and by
    ``finish(sequence)``. ``pages`` is how many there are in each layer's cache;
    ``begin`` raises ValueError, and changes nothing, when they do not suffice.

    A step that checks drafted tokens is ``begin(new, parents)``, ``attend`` in every
    layer, with the positions of ``tree.positions``, and after ``verify_drafts``
    ``keep(path, counts)``. ``fork(sequence, into)`` continues a sequence in two ways: the
    pages stay one until either of them writes to one, which ``begin`` copies first.

    ``axes`` (with theta, pairing and joint) turns Q and K by ``rotary``; without it
    they are used as they come.

    A step cannot be captured into a graph: ``begin`` makes a new page table each
    time, which a replay would not follow. Programs that capture steps keep a page
    table of their own and call ``append_cache`` and ``chunk_attention``.
    """

    def __init__(self, layers: int, sequences: int, heads: int, pages: int, page_tokens: int, *, dim: int = 128,
                 window: int | None = None, sinks: int = 0, frame: int = 1, axes=None, theta: float = 10000.0,
                 pairing: str = "adjacent", joint: bool = False, scale: float | None = None, dtype=torch.bfloat16,
                 device="cuda"):
        if layers < 1 or sequences < 1 or heads < 1 or pages < 1:
            raise ValueError("layers, sequences, heads and pages must be positive")
        if page_tokens < 8 or page_tokens % 8:
            raise ValueError("pages must hold a positive multiple of 8 tokens")
        if dim not in (64, 128) or dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("streaming attention requires head_dim 64 or 128 in BF16 or FP16")
        self.scale = _check_window(window, scale, dim)
        _, self.sinks, self.frame = _mask(window, sinks, frame)
        self.window = window
        self.axes, self.turn = axes, dict(theta=theta, pairing=pairing, joint=joint)
        self.page_tokens, self.device = page_tokens, torch.device(device)
        # All layers' caches, for the operators that take them at once, and each layer's part. To autograd
        # a part is a tensor of its own (.data), which writes to other layers leave as it was.
        shape = (layers, pages, heads, page_tokens, dim)
        self._all = PagedCache(*(torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(2)))
        self.caches = [PagedCache(self._all.k[layer].data, self._all.v[layer].data) for layer in range(layers)]
        self.device = self._all.k.device  # with its index: other devices may become the current one
        self.free = list(range(pages - 1, -1, -1))
        self.owners = [0] * pages        # of each page: the sequences that hold it
        self.tokens = [0] * sequences    # of each sequence, with those of the step that began last
        self.new = [0] * sequences       # of each sequence: those of that step
        self.held = [{} for _ in range(sequences)]  # of each sequence: place in its table -> page
        self.step_tokens = 0
        self.page_table = self.lengths = self.offsets = self.tree = None

    def _behind(self, first: int) -> range:
        """The places of a sequence's table that queries from position ``first`` on do not see."""
        if self.window is None:
            return range(0)
        low = max(0, first // self.frame - int(self.window) + 1) * self.frame
        sinks = min(self.sinks * self.frame, low)
        return range(-(-sinks // self.page_tokens), low // self.page_tokens)

    def _refuse_capture(self) -> None:
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise ValueError("steps of StreamingAttention cannot be captured: the next one has another page table")

    def _writes_all(self) -> None:
        """Tells autograd of a write to all layers."""
        _writes("StreamingAttention", *(t for cache in self.caches for t in cache))

    def _release(self, page: int) -> None:
        self.owners[page] -= 1
        if not self.owners[page]:
            self.free.append(page)

    def begin(self, new, parents=None) -> None:
        """Starts a step of new[s] more tokens in sequence s. ``parents``, of a step of drafts: for each sequence the
        places that its tokens follow, as in ``draft_tree``; ``keep`` ends such a step."""
        self._refuse_capture()
        if self.tree is not None:
            raise ValueError("keep comes before the step after drafts")
        new = [int(n) for n in new]
        if len(new) != len(self.tokens) or min(new) < 0:
            raise ValueError(f"new must give the new tokens of {len(self.tokens)} sequences")
        if parents is not None:
            parents = [[int(p) for p in its] for its in parents]
            if [len(its) for its in parents] != new:
                raise ValueError("parents must give a place for each of the sequences' new tokens")
            if any(not -1 <= p < i for its in parents for i, p in enumerate(its)):
                raise ValueError("a parent must come before the token that follows it, or be -1")
        total = [t + n for t, n in zip(self.tokens, new)]
        gone, wanted, owners = [], [], {}  # owners: of pages that lose some
        steps = [(s, n, length) for s, (n, length) in enumerate(zip(new, total)) if n]
        for s, n, length in steps:
            behind = self._behind(length - n)
            for i, page in self.held[s].items():
                if i in behind:
                    gone.append((s, i))
                    owners[page] = owners.get(page, self.owners[page]) - 1
        for s, n, length in steps:
            for i in range((length - n) // self.page_tokens, -(-length // self.page_tokens)):
                page = self.held[s].get(i)
                if page is None:
                    wanted.append((s, i))
                elif owners.get(page, self.owners[page]) > 1:  # another sequence's too: this one gets a copy
                    wanted.append((s, i))
                    owners[page] = owners.get(page, self.owners[page]) - 1
        free = len(self.free) + sum(not left for left in owners.values())
        if len(wanted) > free:
            raise ValueError(f"{len(wanted)} more pages are needed, {free} are free")
        if any(i in self.held[s] for s, i in wanted):  # copied below
            self._writes_all()
        for s, i in gone:
            self._release(self.held[s].pop(i))
        moves = []
        for s, i in wanted:
            page = self.free.pop()
            if i in self.held[s]:
                moves.append((self.held[s][i], page))
                self._release(self.held[s][i])
            self.held[s][i] = page
            self.owners[page] = 1
        if moves:
            copy_pages(self._all, moves)
        self.tokens, self.new, self.step_tokens = total, new, sum(new)
        width = max(1, max(-(-length // self.page_tokens) for length in total))
        table = [[-1] * width for _ in total]
        for row, held in zip(table, self.held):
            for i, page in held.items():
                row[i] = page
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        values = [table, total, offsets]
        if parents is not None:
            values.append([p for its in parents for p in its])
        self.page_table, self.lengths, self.offsets, *rest = (
            torch.tensor(value, dtype=torch.int32, pin_memory=True).to(self.device, non_blocking=True) for value in values)
        if rest:
            self.tree = draft_tree(*rest, self.lengths, self.offsets)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None = None, *,
               return_lse: bool = False):
        """The layer's attention of the step's new tokens, packed one sequence behind the
        other: q [T, H, D], k and v [T, heads, D]; positions [T, axes] where axes were
        given. Returns o [T, H, D] (and lse [T, H])."""
        if self.offsets is None:
            raise ValueError("attend comes after begin")
        self._refuse_capture()
        if any(t.ndim != 3 or t.shape[0] != self.step_tokens for t in (q, k, v)):
            raise ValueError(f"Q, K and V must be the step's {self.step_tokens} packed tokens [T,H,D]")
        if self.axes is not None:
            if positions is None:
                raise ValueError("positions are needed to turn Q and K")
            q, k = (t[0].transpose(0, 1) for t in rotary(*(t.transpose(0, 1)[None] for t in (q, k)), positions, self.axes, **self.turn))
        cache = append_cache(self.caches[layer], k, v, self.page_table, self.lengths, self.offsets)
        how = dict(window=self.window, sinks=self.sinks, frame=self.frame, scale=self.scale, return_lse=return_lse)
        where = (q, cache, self.page_table, self.lengths, self.offsets)
        return chunk_attention(*where, **how) if self.tree is None else tree_attention(*where, self.tree, **how)

    def keep(self, path: torch.Tensor, counts: torch.Tensor) -> list:
        """Ends a step whose tokens were drafts: of sequence s only the counts[s] at the places path says stay
        (``verify_drafts``' path and counts). Returns the counts as a list, for which it waits for the device."""
        if self.offsets is None:
            raise ValueError("keep comes after begin")
        self._refuse_capture()
        if counts.shape != (len(self.new),) or path.shape != (self.step_tokens,):
            raise ValueError(f"path [{self.step_tokens}] and counts [{len(self.new)}] must be of the step's tokens")
        kept = counts.tolist()
        if any(n and not 0 <= count <= n for count, n in zip(kept, self.new)):
            raise ValueError("counts must be from 0 to the sequences' new tokens")
        _ints("keep", path=path, counts=counts)
        _gpu("keep", self._all.k, path, counts)
        self._writes_all()
        keep_drafts(self._all, self.page_table, self.lengths, self.offsets, path, counts)
        for s, (count, n) in enumerate(zip(kept, self.new)):
            if n:
                self.tokens[s] += count - n
                last = -(-self.tokens[s] // self.page_tokens)
                for i in [i for i in self.held[s] if i >= last]:
                    self._release(self.held[s].pop(i))
        self.new = [0] * len(self.new)
        self.page_table = self.lengths = self.offsets = self.tree = None
        return kept

    def fork(self, sequence: int, into: int) -> None:
        """Continues a sequence in a second way: ``into``, which must be one that has no tokens, gets all that
        ``sequence`` has. No page is copied before one of them writes to it. Between steps: the next call is ``begin``."""
        if self.tree is not None:
            raise ValueError("keep comes before fork")
        if self.tokens[into] or self.held[into]:
            raise ValueError("into must be a sequence without tokens")
        for page in self.held[sequence].values():
            self.owners[page] += 1
        self.held[into] = dict(self.held[sequence])
        self.tokens[into] = self.tokens[sequence]
        self.page_table = self.lengths = self.offsets = None

    def finish(self, sequence: int) -> None:
        """Gives a sequence's pages back, as far as no other one has them; it starts again at position 0."""
        for page in self.held[sequence].values():
            self._release(page)
        self.held[sequence] = {}
        self.tokens[sequence] = self.new[sequence] = 0
