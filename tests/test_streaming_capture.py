"""StreamingAttention inside a graph's capture: refused before anything changes (CPU only)."""
import pytest
import torch

from ab_attention.streaming import StreamingAttention


def test_steps_are_not_captured(monkeypatch):
    stream = StreamingAttention(1, 2, 1, 4, 16, dim=64, device="cpu")
    stream.device = torch.device("cuda", 0)
    x = torch.zeros((3, 1, 64), dtype=torch.bfloat16)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    before = (list(stream.free), list(stream.tokens), [dict(h) for h in stream.held])
    with pytest.raises(ValueError, match="captured"):
        stream.begin([3, 0])
    assert before == (stream.free, stream.tokens, stream.held) and stream.offsets is None
    stream.offsets, stream.step_tokens = torch.zeros(3, dtype=torch.int32), 3
    with pytest.raises(ValueError, match="captured"):
        stream.attend(0, x, x, x)
    stream.finish(0)  # touches no tensor
