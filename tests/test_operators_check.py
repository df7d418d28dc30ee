"""Which device check_operators looks at (CPU: the device calls are stand-ins)."""
import pytest
import torch

from boonta_b200 import _lib


@pytest.fixture
def looked_at(monkeypatch):
    seen = []

    class Device:
        def __init__(self, index):
            seen.append(index)

        def __enter__(self):
            return 0

        def __exit__(self, *exc):
            pass

    class Library:
        @staticmethod
        def bt_operators_check(stream):
            return _lib.BT_OK

    monkeypatch.setattr(_lib, "on_device", Device)
    monkeypatch.setattr(_lib, "lib", lambda: Library)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    return seen


@pytest.mark.parametrize("device,index", [(None, 3), ("cuda", 3), (torch.device("cuda"), 3), ("cuda:0", 0),
                                          ("cuda:5", 5), (torch.device("cuda", 2), 2), (1, 1), (0, 0)])
def test_the_device_that_is_checked(looked_at, device, index):
    _lib.check_operators(device)
    assert looked_at == [index]


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), "meta"])
def test_only_cuda_devices_are_checked(looked_at, device):
    with pytest.raises(ValueError, match="CUDA"):
        _lib.check_operators(device)
    assert not looked_at
