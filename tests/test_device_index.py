"""device_index, the tensors' check of the calls whose host time matters (no GPU: stand-ins for tensors)."""
import pytest

from mfd_b200 import _lib


class _On:
    def __init__(self, index):
        self.index = index

    def get_device(self):
        return self.index


def test_the_device_all_tensors_share(monkeypatch):
    monkeypatch.setattr(_lib, "_current_device", lambda: 1, raising=False)
    assert _lib.device_index(_On(1), _On(1), None, _On(1)) == 1


def test_tensors_of_a_device_that_is_not_current_are_refused(monkeypatch):
    """The kernel would run on the current device, and read memory of another."""
    monkeypatch.setattr(_lib, "_current_device", lambda: 0, raising=False)
    with pytest.raises(RuntimeError, match="cuda:1.*cuda:0"):
        _lib.device_index(_On(1), _On(1))
