"""Workspace, the scratch that calls outside of CUDA graphs share, on the host (no GPU)."""
import weakref

import pytest
import torch

from mfd_b200 import _lib
from mfd_b200._lib import Workspace

DEV = torch.device("cpu", 0)


@pytest.fixture(autouse=True)
def _fresh(monkeypatch):
    monkeypatch.setattr(Workspace, "_cache", {})
    if hasattr(Workspace, "_outgrown"):
        monkeypatch.setattr(Workspace, "_outgrown", [])


@pytest.mark.parametrize("get", [lambda n: Workspace.get(DEV, "attn", n), lambda n: Workspace.tickets(DEV, n)])
def test_a_buffer_that_was_outgrown_stays_allocated(get):
    """A CUDA graph that was captured with it goes on writing to it."""
    small = get(2000)
    address, alive = small.data_ptr(), weakref.ref(small)
    large = get(50000)
    assert large.data_ptr() != address and large.numel() >= 50000
    del small
    assert alive() is not None and alive().data_ptr() == address
    assert get(2000) is large


@pytest.mark.parametrize("get", [lambda n: Workspace.get(DEV, "attn", n), lambda n: Workspace.tickets(DEV, n)])
def test_a_buffer_that_is_made_while_capturing_is_not_kept(monkeypatch, get):
    """It is zeroed by a node of that graph alone, so a plain call, or another graph, must not find it."""
    with monkeypatch.context() as m:
        m.setattr(_lib, "_recording", lambda: True, raising=False)
        assert get(2000).numel() >= 2000 and not get(2000).any()
    assert not Workspace._cache
    plain = get(3000)
    with monkeypatch.context() as m:
        m.setattr(_lib, "_recording", lambda: True, raising=False)
        assert get(2000) is plain  # zeroed before
        assert get(100000) is not plain
    assert get(3000) is plain
