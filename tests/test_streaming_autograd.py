"""What autograd is told of the streaming operators: nothing of theirs is launched here (CPU only)."""
import pytest
import torch
from torch.autograd import forward_ad

from ab_attention import streaming
from ab_attention.streaming import PagedCache, append_cache, chunk_attention, rotary, window_attention

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


_POS = torch.zeros((3, 1), dtype=torch.int32)
_CALLS = [
    lambda x, other: rotary(x, other, _POS, (64,)),
    lambda x, other: rotary(other, x, _POS, (64,)),
    lambda x, other: rotary(other, None, x[0, 0, :, :1].float(), (64,)),
    lambda x, other: window_attention(x, other, other),
    lambda x, other: window_attention(other, x, other, return_lse=True),
    lambda x, other: window_attention(other, other, x),
    lambda x, other: chunk_attention(x[0], PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64)), *_where()),
    lambda x, other: chunk_attention(other[0], PagedCache(_x(2, 3, 8, 64), x.new_zeros(2, 3, 8, 64) + x[0, 0, 0]), *_where()),
    lambda x, other: append_cache(PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64)), x[0], other[0], *_where()),
    lambda x, other: append_cache(PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64)), other[0], x[0], *_where()),
]


@pytest.mark.parametrize("call", _CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(no_launch, call, grad):
    """A tangent that the kernels cannot follow raises; without one, and inside a level, the calls run."""
    x, other = _x(1, 3, 3, 64), _x(1, 3, 3, 64).requires_grad_(grad)
    call(x, other)
    with forward_ad.dual_level():
        call(x, other)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            call(dual, other)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            call(dual, other)


@pytest.mark.parametrize("op", [lambda x: rotary(x, None, _POS, (64,))[0], lambda x: window_attention(x, x, x),
                                lambda x: window_attention(x, x, x, return_lse=True)[1]])
def test_forward_mode_over_a_gradient_is_refused(no_launch, op):
    x = _x(1, 3, 3, 64).requires_grad_()
    out = op(x)
    with forward_ad.dual_level():
        weight = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad((out * weight).sum(), x)


def test_writes_are_counted(no_launch):
    """The caches' and out's versions, those of their bases and views with them; tensors of inference mode have none."""
    base = _x(2, 2, 3, 8, 64)
    cache, x, out = PagedCache(base[:, 0], base[:, 1]), _x(3, 3, 64), _x(3, 3, 64)
    versions = lambda *tensors: [t._version for t in tensors]  # noqa: E731
    before = versions(base, cache.k, cache.v)
    append_cache(cache, x, x, *_where())
    assert all(a > b for a, b in zip(versions(base, cache.k, cache.v), before))
    before = versions(base, x)
    chunk_attention(x, cache, *_where())
    assert versions(base, x, out) == [*before, 0]
    assert chunk_attention(x, cache, *_where(), out=out) is out and out._version == 1 and versions(base, x) == before
    with torch.inference_mode():
        cache, out = PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64)), _x(3, 3, 64)
        append_cache(cache, x, x, *_where())
    with torch.no_grad():
        append_cache(cache, x, x, *_where())
        chunk_attention(x, cache, *_where(), out=out)


def test_tensors_that_require_a_gradient_are_not_written(no_launch):
    x, cache = _x(3, 3, 64), PagedCache(_x(2, 3, 8, 64), _x(2, 3, 8, 64))
    for out in (_x(3, 3, 64).requires_grad_(), _x(3, 3, 64).requires_grad_() * 2):
        with pytest.raises(ValueError, match="requires a gradient"):
            chunk_attention(x, cache, *_where(), out=out)
    learned = PagedCache(cache.k, _x(2, 3, 8, 64).requires_grad_())
    with pytest.raises(ValueError, match="requires a gradient"):
        append_cache(learned, x, x, *_where())
    with torch.no_grad():
        append_cache(learned, x, x, *_where())
    assert not chunk_attention(x.clone().requires_grad_(), learned, *_where()).requires_grad
