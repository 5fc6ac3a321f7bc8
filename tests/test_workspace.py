"""Workspace, the scratch that calls outside of CUDA graphs share, on the host (no GPU)."""
import weakref

import pytest
import torch

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
