"""
_lib.stream_of without a GPU: it names the device whose stream it returns by everything that torch.cuda.current_stream takes, and refuses
what that refuses.
"""
import pytest
import torch

from igs_b200 import _lib


@pytest.fixture
def handles(monkeypatch):
    """Device i's stream handle is 100 + i; device 2 is the current one."""
    monkeypatch.setattr(_lib, "raw_stream_of", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)


@pytest.mark.parametrize("device,index", [(None, 2), ("cuda", 2), (torch.device("cuda"), 2), (0, 0), (1, 1), (3, 3), ("cuda:1", 1),
                                          (torch.device("cuda", 0), 0), (torch.device("cuda", 3), 3)])
def test_stream_of_the_device_named(handles, device, index):
    assert _lib.stream_of(device).value == 100 + index


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), torch.device("meta"), "gpu:0", 1.0, object(), -1])
def test_stream_of_refuses(handles, device):
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        _lib.stream_of(device)
