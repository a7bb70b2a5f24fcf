"""_lib.current asks for the stream of the tensor's device, and whether that one is captured, whichever device is current."""
import pytest
import torch

from came_amd import _lib


class OnGpu(torch.Tensor):
    """A tensor that says it lies on GPU `at`."""

    at = 0
    is_cuda = True

    def get_device(self):
        return self.at

    @property
    def device(self):
        return torch.device("cuda", self.at)


@pytest.mark.parametrize("captured", [0, 1, None])
@pytest.mark.parametrize("at,now", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_the_tensors_device_is_asked(monkeypatch, at, now, captured):
    current = [now]

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.was, current[0] = current[0], self.device

        def __exit__(self, *_):
            current[0] = self.was

    monkeypatch.setattr(_lib, "_raw_stream", lambda d: 100 + d)
    monkeypatch.setattr(_lib, "_current_device", lambda: current[0])
    monkeypatch.setattr(_lib, "_Device", Device)
    monkeypatch.setattr(_lib, "_capturing", lambda: current[0] == captured)
    t = torch.zeros(2).as_subclass(OnGpu)
    t.at = at
    assert _lib.current(t) == (100 + at, captured == at)
    assert current == [now]


def test_what_is_on_no_gpu():
    assert _lib.current(torch.zeros(2)) == _lib.current(None) == (0, False)
