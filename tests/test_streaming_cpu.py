"""What the streaming operators refuse, before any launch (CPU only)."""
import ctypes

import pytest
import torch

from ab_attention import _lib
from ab_attention.streaming import (PagedCache, StreamingAttention, append_cache, chunk_attention, rotary,
                                    window_attention)

BF16 = torch.bfloat16


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


_POS = torch.zeros((5, 3), dtype=torch.int32)


@pytest.mark.parametrize("args,kw,msg", [
    ((_z(2, 5, 128), None, _POS, (44, 42, 42)), {}, "B,H,N,D"),
    ((_z(1, 2, 5, 128), _z(1, 2, 6, 128), _POS, (44, 42, 42)), {}, "same batch"),
    ((_z(1, 2, 5, 128), _z(1, 2, 5, 128, dtype=torch.float16), _POS, (44, 42, 42)), {}, "one type"),
    ((_z(1, 2, 5, 128, dtype=torch.float64), None, _POS, (44, 42, 42)), {}, "BF16"),
    ((_z(1, 2, 5, 12), None, _POS, (4, 4, 4)), {}, "multiple of 8"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 44)), {}, "add up"),
    ((_z(1, 2, 5, 128), None, _POS, (43, 42, 42)), {}, "even"),
    ((_z(1, 2, 5, 128), None, _POS, ()), {}, "1 to 4"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 42)), {"pairing": "other"}, "pairing"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 40)), {"pairing": "halves"}, "multiple of 16"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 42)), {"theta": 0.0}, "theta"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 42)), {"theta": float("inf")}, "theta"),
    ((_z(1, 2, 5, 128), None, _POS.double(), (44, 42, 42)), {}, "int32"),
    ((_z(1, 2, 5, 128), None, _POS[:4], (44, 42, 42)), {}, "positions must be"),
    ((_z(2, 2, 5, 128), None, _POS[None].expand(3, 5, 3), (44, 42, 42)), {}, "positions must be"),
    ((_z(1, 2, 5, 128), None, _POS, (44, 42, 42)), {}, "CUDA"),
])
def test_rotary_refuses(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        rotary(*args, **kw)


@pytest.mark.parametrize("q,k,kw,msg", [
    (_z(2, 8, 64), _z(2, 8, 64), {}, "B,H,N,D"),
    (_z(1, 2, 8, 64), _z(1, 2, 9, 64), {}, "share"),
    (_z(1, 2, 8, 96), _z(1, 2, 8, 96), {}, "64 or 128"),
    (_z(1, 2, 8, 64, dtype=torch.float32), _z(1, 2, 8, 64, dtype=torch.float32), {}, "BF16"),
    (_z(1, 3, 8, 64), _z(1, 2, 8, 64), {}, "multiple"),
    (_z(1, 2, 8, 64), _z(1, 0, 8, 64), {}, "multiple"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"window": 0}, "window"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"window": -3}, "window"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"sinks": -1}, "sinks"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"frame": 0}, "frame"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"scale": float("nan")}, "scale"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"lengths": torch.zeros(2, dtype=torch.int32)}, "lengths"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {"lengths": torch.zeros(1, dtype=torch.int64)}, "lengths"),
    (_z(1, 2, 8, 64), _z(1, 2, 8, 64), {}, "CUDA"),
])
def test_window_attention_refuses(q, k, kw, msg):
    with pytest.raises(ValueError, match=msg):
        window_attention(q, k, k, **kw)


def _cache(pages=4, heads=2, page=16, dim=64, dtype=BF16):
    return PagedCache(_z(pages, heads, page, dim, dtype=dtype), _z(pages, heads, page, dim, dtype=dtype))


_TABLE, _LENGTHS, _OFFSETS = (torch.zeros(s, dtype=torch.int32) for s in ((2, 3), (2,), (3,)))


@pytest.mark.parametrize("change,msg", [
    (dict(q=_z(1, 5, 2, 64)), r"T,H,D"),
    (dict(cache=_cache(dim=128)), "cache must be"),
    (dict(cache=PagedCache(_z(4, 2, 16, 64), _z(4, 2, 8, 64))), "cache must be"),
    (dict(cache=_cache(dtype=torch.float16)), "same type"),
    (dict(cache=_cache(page=12)), "multiple of 8"),
    (dict(cache=_cache(page=0)), "multiple of 8"),
    (dict(cache=PagedCache(_z(4, 2, 64, 16).transpose(2, 3), _z(4, 2, 16, 64))), "rows must be"),
    (dict(cache=_cache(heads=3)), "multiple"),
    (dict(page_table=torch.zeros((3, 3), dtype=torch.int32)), "one batch"),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), "one batch"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "int32"),
    (dict(page_table=torch.zeros((3, 2), dtype=torch.int32).T), "contiguous int32"),
    (dict(), "CUDA"),
])
def test_cache_operators_refuse(change, msg):
    how = dict(q=_z(5, 2, 64), cache=_cache(), page_table=_TABLE, lengths=_LENGTHS, offsets=_OFFSETS)
    how.update(change)
    q = how.pop("q")
    with pytest.raises(ValueError, match=msg):
        chunk_attention(q, **how)
    with pytest.raises(ValueError, match=msg):
        append_cache(how["cache"], q, q, how["page_table"], how["lengths"], how["offsets"])


def test_append_refuses_other_shapes():
    with pytest.raises(ValueError, match="one shape"):
        append_cache(_cache(), _z(5, 2, 64), _z(4, 2, 64), _TABLE, _LENGTHS, _OFFSETS)


_A = 4096  # a 16-byte aligned stand-in address: every case is refused before any runtime call


def _window_args(**change):
    a = _lib.WindowArgs(q=_A, k=_A, v=_A, out=_A, batch=1, heads=2, kv_heads=1, tokens=8, dim=64, dtype=0, window=0, sinks=0,
                        frame=1, scale=0.1, pages=4, page_tokens=16, table_width=2)
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        setattr(a, name, (ctypes.c_int64 * 3)(1024, 512, 64))
    for name, value in change.items():
        setattr(a, name, (ctypes.c_int64 * 3)(*value) if name.endswith("stride") else value)
    return a


@pytest.mark.parametrize("change,msg", [
    (dict(heads=3, kv_heads=2), b"multiple of kv_heads"), (dict(dim=96), b"64 or 128"), (dict(dtype=2), b"bf16 or fp16"),
    (dict(frame=0), b"frame"), (dict(window=-1), b"negative"), (dict(scale=float("inf")), b"finite"),
    (dict(tokens=1 << 30), b"too many"), (dict(batch=70000), b"too many"), (dict(k_stride=(1024, 512, 12)), b"strides"),
    (dict(q_stride=(1024, -8, 64)), b"strides"), (dict(tokens=1 << 25, k_stride=(1 << 31, 1 << 31, 64)), b"4 GiB"),
    (dict(q=0), b"null"), (dict(out=0), b"null"), (dict(k=_A + 8), b"aligned"), (dict(out=_A + 4), b"aligned"),
])
def test_window_entry_refuses(change, msg):
    lib = _lib.load()
    assert lib.ab_window_attention(_window_args(**change), None) == 1
    assert msg in lib.ab_last_error() and lib.ab_last_error().startswith(b"window_attention:")


@pytest.mark.parametrize("change,msg", [
    (dict(page_tokens=12), b"multiple of 8"), (dict(page_tokens=0), b"multiple of 8"), (dict(lengths=0), b"null"),
    (dict(table_width=1 << 28), b"fewer than 2^30"), (dict(pages=-1), b"pages"), (dict(k=0), b"null"),
    (dict(page_tokens=1 << 22, k_stride=(0, 0, 1024)), b"4 GiB"),
])
def test_chunk_entry_refuses(change, msg):
    lib = _lib.load()
    args = _window_args(**{**dict(lengths=_A, offsets=_A, page_table=_A), **change})
    assert lib.ab_chunk_attention(args, None) == 1
    assert msg in lib.ab_last_error()


def test_entries_of_nothing_launch_nothing():
    lib = _lib.load()
    assert lib.ab_window_attention(_window_args(tokens=0), None) == 0
    assert lib.ab_window_attention(_window_args(batch=0), None) == 0
    assert lib.ab_window_workspace_bytes(_window_args(tokens=0)) == 0
    assert lib.ab_window_workspace_bytes(None) == 0
    assert lib.ab_window_attention(None, None) == 1 and b"null" in lib.ab_last_error()
    assert lib.ab_rotary(None, None) == 1 and lib.ab_append_cache(None, None) == 1


def test_workspace_of_a_split_call():
    """Few rows over many keys are split; the workspace holds each part's float32 rows, sums and references."""
    lib = _lib.load()
    args = _window_args(lengths=_A, offsets=_A, page_table=_A, tokens=1, batch=1, table_width=2048)
    size = lib.ab_window_workspace_bytes(args)
    row = 2 * (64 * 4 + 8)
    assert size > 0 and size % row == 0 and size // row <= 2048 * 16 // 32
    assert lib.ab_window_workspace_bytes(_window_args(tokens=100000, q_stride=(0, 0, 64), heads=64)) == 0


def _grad_args(**change):
    g = _lib.WindowGradArgs(dout=_A, dq=_A, dk=_A, dv=_A)
    g.forward = _window_args(lse=_A, workspace=_A, workspace_bytes=1 << 20)
    for name in ("dout_stride", "dq_stride", "dk_stride", "dv_stride"):
        setattr(g, name, (ctypes.c_int64 * 3)(1024, 512, 64))
    for name, value in change.items():
        target = g.forward if hasattr(g.forward, name) else g
        setattr(target, name, (ctypes.c_int64 * 3)(*value) if name.endswith("stride") else value)
    return g


@pytest.mark.parametrize("change,msg", [
    (dict(dout=0), b"null"), (dict(dk=0), b"null"), (dict(lse=0), b"null"), (dict(workspace=0), b"null"),
    (dict(dq=_A + 8), b"aligned"), (dict(out=_A + 8), b"aligned"), (dict(out_rest=_A + 8), b"aligned"), (dict(workspace_bytes=64), b"smaller"),
    (dict(dv_stride=(1024, 512, 4)), b"strides"), (dict(out_stride=(1024, 512, 68)), b"strides"), (dict(dim=32), b"64 or 128"),
])
def test_gradient_entry_refuses(change, msg):
    lib = _lib.load()
    assert lib.ab_window_attention_grad(_grad_args(**change), None) == 1
    assert msg in lib.ab_last_error() and lib.ab_last_error().startswith(b"window_attention_grad:")


def test_gradient_workspace():
    """Normalisers and deltas of every 32 queries; float32 parts only where sinks are seen from far behind a window."""
    lib = _lib.load()
    assert lib.ab_window_grad_workspace_bytes(_grad_args(tokens=0)) == 0
    strides = dict(q_stride=(1 << 22, 1 << 20, 64), k_stride=(1 << 22, 1 << 20, 64), v_stride=(1 << 22, 1 << 20, 64))
    plain = lib.ab_window_grad_workspace_bytes(_grad_args(tokens=1024, window=100, **strides))
    assert plain == 2 * 32 * 64 * 4
    sinks = lib.ab_window_grad_workspace_bytes(_grad_args(tokens=1024, window=100, sinks=4, **strides))
    assert (sinks - plain) % (2 * 128 * 64 * 4) == 0 and sinks > plain
    far = dict(q_stride=(0, 1 << 20, 64), k_stride=(0, 1 << 20, 64), v_stride=(0, 1 << 20, 64), batch=1)
    big = lib.ab_window_grad_workspace_bytes(_grad_args(tokens=1 << 20, window=1, sinks=1 << 19, **far))
    assert 0 < big <= (1 << 30) + 2 * (1 << 15) * 256


def test_rows_out_of_reach_are_copied():
    """Heads of which a kernel's 32-bit offsets do not reach the last row are read from a copy."""
    from ab_attention.streaming import _strided

    base = torch.zeros(64, dtype=BF16)
    near = base.as_strided((1, 1, 1000, 64), (0, 0, 0, 1))
    assert _strided(near) is near
    far = torch.empty((1, 1, 70, 64), dtype=BF16, device="meta").as_strided((1, 1, 70, 64), (1 << 36, 1 << 36, 1 << 25, 1))
    assert far.stride(2) * (70 + 64) >= (1 << 31) and _strided(far).is_contiguous()
    packed = torch.empty((70, 2, 64), dtype=BF16, device="meta").as_strided((70, 2, 64), (1 << 27, 64, 1))
    assert _strided(packed) is packed


@pytest.mark.parametrize("change,msg", [(dict(layers=0), "positive"), (dict(pages=0), "positive"), (dict(page_tokens=12), "multiple of 8"),
                                        (dict(dim=96), "64 or 128"), (dict(dtype=torch.float32), "BF16"), (dict(window=0), "window"),
                                        (dict(frame=0), "frame"), (dict(sinks=-1), "sinks")])
def test_streaming_attention_refuses(change, msg):
    how = dict(layers=1, sequences=1, heads=1, pages=2, page_tokens=16, device="cpu")
    how.update(change)
    with pytest.raises(ValueError, match=msg):
        StreamingAttention(**how)


def test_streaming_attention_needs_a_step_and_positions():
    stream = StreamingAttention(1, 1, 1, 2, 16, dim=64, device="cpu", axes=(64,))
    x = _z(3, 1, 64)
    with pytest.raises(ValueError, match="begin"):
        stream.attend(0, x, x, x)
    stream.offsets, stream.step_tokens = _OFFSETS, 3
    with pytest.raises(ValueError, match="positions"):
        stream.attend(0, x, x, x)
    with pytest.raises(ValueError, match="3 packed tokens"):
        stream.attend(0, x[:2], x, x)


def test_pages_behind_the_window():
    """Pages go back when none of their tokens can be seen again, whatever the sizes of frames and pages."""
    from streaming_reference import seen_mask

    for window, sinks, frame, page in ((3, 1, 10, 8), (1, 0, 7, 16), (40, 5, 1, 8), (2, 2, 24, 8), (2, 1, 8, 24)):
        stream = StreamingAttention(1, 1, 1, 2, page, dim=64, window=window, sinks=sinks, frame=frame, device="cpu")
        keys = torch.arange(400)
        for first in (0, 1, 39, 40, 41, 200, 399):
            seen = seen_mask(torch.arange(first, 400), keys, window, sinks, frame).any(0)
            behind = stream._behind(first)
            for i in range(400 // page):
                inside = seen[i * page:(i + 1) * page]
                if i in behind:
                    assert not inside.any()
                elif (i + 1) * page <= first // frame * frame:  # a page of the past that is kept holds something to see
                    assert inside.any(), (window, sinks, frame, page, first, i)
