"""Which device a call makes current: that of its first tensor on a GPU, whatever
comes before it.  Tensors that only look as if they were on one (no GPU here)."""
import pytest
import torch

from surfface_hip import _torch as T
from surfface_hip.scores import Int8Rows


@pytest.fixture
def device(monkeypatch):
    """Tensors of another device than the current one, and what the calls made current."""
    made = []

    class Current:
        def __init__(self, what):
            self.what = what

        def __enter__(self):
            made.append(self.what)

        def __exit__(self, *exc):
            pass

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: Current(s.device))
    return made


def fake(index):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        return torch.empty(4, 16, device=f"cuda:{index}")


class Stream:
    def __init__(self, index):
        self.device = torch.device("cuda", index)


@pytest.mark.parametrize("wrap", [T.enqueues, T.on_device])
def test_the_first_tensor_decides(device, wrap):
    call = wrap(lambda *a, **k: "done")
    q = fake(1)
    rows = Int8Rows(q, q, 16)
    for args, kwargs in (((q,), {}), ((2.0, q), {}), ((), {"scale": 2.0, "queries": q}), ((None, "mean", rows), {}),
                         ((), {"dtype": torch.float32, "items": rows}), ((torch.zeros(3), q), {})):
        del device[:]
        assert call(*args, **kwargs) == "done"
        assert device == [torch.device("cuda", 1)], (args, kwargs)
    del device[:]
    assert call(scale=2.0, queries=fake(0)) == call(torch.zeros(3)) == call() == "done"
    assert not device


def test_a_stream_of_another_device(device):
    call = T.enqueues(lambda *a, **k: "done")
    for kwargs in ({"scale": 2.0, "queries": fake(0)}, {"queries": fake(0), "scale": 2.0}):
        with pytest.raises(ValueError, match="stream is on"):
            call(stream=Stream(1), **kwargs)
    with pytest.raises(ValueError, match="stream is on"):
        call(2.0, Int8Rows(fake(0), fake(0), 16), stream=Stream(1))
    assert not device
