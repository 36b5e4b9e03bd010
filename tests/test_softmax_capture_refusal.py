"""The backward pass of a loss that was computed before the capture began is refused
before any work (no GPU here, so the capture is the test's word)."""
import pytest
import torch

from surfface_hip import softmax


class Context:
    saved_tensors, of, needs_input_grad = (), (None,) * 5, (True, True)


def test_backward_in_a_capture(monkeypatch):
    monkeypatch.setattr(softmax, "_backward", lambda *a: pytest.fail("backward ran"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="graph capture"):
        softmax._SoftmaxLoss.backward(Context(), torch.zeros(()))
