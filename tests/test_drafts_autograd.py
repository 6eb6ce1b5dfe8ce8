"""What autograd is told of the caches that StreamingAttention writes: nothing is launched here (CPU only)."""
import pytest
import torch

from ab_attention import streaming
from ab_attention.streaming import StreamingAttention


@pytest.fixture
def stream(monkeypatch):
    """Three layers on the CPU, two sequences that share a page, without the operators' launches."""
    monkeypatch.setattr(streaming, "_gpu", lambda name, first, *others: first.device)
    monkeypatch.setattr(streaming, "_call", lambda *args: None)
    monkeypatch.setattr(streaming, "_run", lambda *args: None)
    tensor = torch.tensor
    monkeypatch.setattr(torch, "tensor", lambda values, dtype, pin_memory: tensor(values, dtype=dtype))
    stream = StreamingAttention(3, 2, 1, 6, 8, dim=64, device="cpu")
    stream.begin([5, 0])
    stream.fork(0, 1)
    return stream


def _saved(stream, layer):
    """A loss whose gradient needs the layer's keys and values as they are."""
    x = torch.ones(64, dtype=torch.bfloat16, requires_grad=True)
    cache = stream.caches[layer]
    return (x * cache.k).sum() + (x * cache.v).sum()


def _attend(stream, layer):
    x = torch.zeros((stream.step_tokens, 1, 64), dtype=torch.bfloat16)
    stream.attend(layer, x, x, x)


def test_a_layer_is_written_alone(stream):
    stream.finish(1)
    stream.begin([2, 0])
    losses = [_saved(stream, layer) for layer in range(3)]
    _attend(stream, 1)
    losses[0].backward()
    losses[2].backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        losses[1].backward()


def test_pages_are_copied_in_all_layers(stream):
    losses = [_saved(stream, layer) for layer in range(3)]
    stream.begin([0, 1])  # the page that both have is copied
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    losses = [_saved(stream, layer) for layer in range(3)]
    stream.begin([1, 1])  # nothing is
    for loss in losses:
        loss.backward()


def test_drafts_are_kept_in_all_layers(stream):
    stream.begin([3, 0], [[-1, 0, 0], []])
    losses = [_saved(stream, layer) for layer in range(3)]
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32"):
        stream.keep(ints.long(), ints[:2])
    losses.pop().backward()  # a refused call writes nothing
    assert stream.keep(ints, ints[:2]) == [0, 0]
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_layers_that_learn_are_not_written(stream):
    """As append_cache refuses it; a step that is refused changes nothing."""
    stream.caches[2].v.requires_grad_()
    before = (list(stream.free), list(stream.owners), list(stream.tokens), [dict(held) for held in stream.held])
    with pytest.raises(ValueError, match="requires a gradient"):
        stream.begin([0, 1])
    assert before == (stream.free, stream.owners, stream.tokens, stream.held)
    stream.finish(1)
    stream.begin([3, 0], [[-1, 0, 0], []])
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="requires a gradient"):
        stream.keep(ints, ints[:2])
    with torch.no_grad():
        assert stream.keep(ints, ints[:2]) == [0, 0]


def test_all_layers_are_reached(stream):
    """The operators that take all layers at once reach the tensors that single layers are read from."""
    taken = []
    pack = streaming._COPY.pack
    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(streaming, "_COPY", type("", (), dict(pack=lambda *args: (taken.append(args), pack(*args))[1])))
        stream.begin([0, 1])
    (k, v, _, count, layers, *_), = taken
    strides = taken[0][9:11]
    assert (count, layers) == (1, 3)
    for layer, cache in enumerate(stream.caches):
        assert cache.k.data_ptr() == k + 2 * layer * strides[0] and cache.v.data_ptr() == v + 2 * layer * strides[1]
        assert cache.k.shape == (6, 1, 8, 64) and cache.k.is_contiguous() and cache.v.is_contiguous()


def test_steps_in_inference_mode(monkeypatch, stream):
    """Caches of inference mode have no version to be counted, others are counted there too."""
    before = [t._version for cache in stream.caches for t in cache]
    with torch.inference_mode():
        stream.begin([0, 1])
        other = StreamingAttention(2, 2, 1, 6, 8, dim=64, device="cpu")
        other.begin([5, 0])
        other.fork(0, 1)
        other.begin([0, 1])
        _attend(other, 1)
    assert all(t._version > x for x, t in zip(before, (t for cache in stream.caches for t in cache)))
