"""Layouts that the streaming operators take or refuse to write to: nothing of theirs is launched here (CPU only)."""
import pytest
import torch

from ab_attention import streaming
from ab_attention.streaming import PagedCache, append_cache, chunk_attention

BF16 = torch.bfloat16


@pytest.fixture
def no_launch(monkeypatch):
    """The operators' Python side on CPU tensors."""
    monkeypatch.setattr(streaming, "_gpu", lambda name, first, *others: first.device)
    monkeypatch.setattr(streaming, "_call", lambda *args: None)
    monkeypatch.setattr(streaming, "_run", lambda *args: None)


def _x(*shape):
    return torch.zeros(shape, dtype=BF16)


def _where():
    return [torch.zeros(s, dtype=torch.int32) for s in ((1, 2), (1,), (2,))]  # page table, lengths, offsets


@pytest.mark.parametrize("stride,own", [
    ((192, 64, 1), True), ((64, 320, 1), True), ((1024, 128, 1), True), ((68, 400, 1), True), ((320, 64, 1), True),
    ((0, 64, 1), False), ((192, 0, 1), False), ((32, 320, 1), False), ((192, 32, 1), False), ((128, 64, 1), False),
    ((64, 64, 1), False), ((64, 256, 1), False)])
def test_rows_of_out(no_launch, stride, own):
    """out [5, 3, 64]: every row its own, whatever the order of tokens and heads in memory."""
    q, cache = _x(5, 3, 64), PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64))
    out = _x(8192).as_strided((5, 3, 64), stride)
    # Which elements share memory, by counting them.
    at = torch.arange(8192).as_strided((5, 3, 64), stride).reshape(-1)
    assert (at.unique().numel() == at.numel()) == own
    if own:
        assert chunk_attention(q, cache, *_where(), out=out) is out
    else:
        with pytest.raises(ValueError, match="each its own"):
            chunk_attention(q, cache, *_where(), out=out)


@pytest.mark.parametrize("stride,own", [
    ((1536, 512, 64, 1), True), ((1536, 64, 192, 1), True), ((64, 4096, 512, 1), True), ((4096, 1280, 128, 1), True),
    ((1024, 512, 64, 1), False), ((1536, 512, 32, 1), False), ((0, 512, 64, 1), False), ((1536, 0, 64, 1), False)])
def test_rows_of_a_cache(no_launch, stride, own):
    """A cache [2, 3, 8, 64] that is written: views of any order, none whose rows overlap (it may be read)."""
    view = _x(32768).as_strided((2, 3, 8, 64), stride)
    at = torch.arange(32768).as_strided((2, 3, 8, 64), stride).reshape(-1)
    assert (at.unique().numel() == at.numel()) == own
    x = _x(5, 3, 64)
    for cache in (PagedCache(view, _x(2, 3, 8, 64)), PagedCache(_x(2, 3, 8, 64), view)):
        chunk_attention(x, cache, *_where())
        if own:
            assert append_cache(cache, x, x, *_where()) is cache
        else:
            with pytest.raises(ValueError, match="overlap"):
                append_cache(cache, x, x, *_where())


def test_keys_and_values_of_two_devices(monkeypatch):
    monkeypatch.setattr(streaming, "_gpu", lambda name, first, *others: first.device)
    x = _x(5, 3, 64)
    with pytest.raises(ValueError, match="one CUDA device"):
        append_cache(PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64)), x, x.to("meta"), *_where())
