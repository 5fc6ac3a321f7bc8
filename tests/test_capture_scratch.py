"""CaptureScratch, the scratch of calls recorded into CUDA graphs, on the host: what is shared, and what is not (no GPU)."""
import ctypes

import pytest
import torch

from mfd_b200 import _lib
from mfd_b200._lib import CaptureScratch

DEV = torch.device("cpu", 0)


@pytest.fixture(autouse=True, params=["spare tickets", "none"])
def _fresh(monkeypatch, request):
    monkeypatch.setattr(CaptureScratch, "_held", {})
    monkeypatch.setattr(CaptureScratch, "_spare", {})
    if request.param == "spare tickets":
        CaptureScratch.prepare(DEV)


def _bytes(address, n):
    return bytes((ctypes.c_uint8 * n).from_address(address))


def test_calls_of_one_capture_and_stream_share_their_scratch():
    a = CaptureScratch.get(DEV, "attn", 7, 1, 5000, 10)
    assert CaptureScratch.get(DEV, "attn", 7, 1, 4000, 10) == a
    assert a[1] >= 5000 and a[3] >= 10 and _bytes(a[2], 4 * a[3]) == bytes(4 * a[3])


def test_captures_streams_and_purposes_have_their_own():
    get = CaptureScratch.get
    kept = [get(DEV, "attn", 7, 1, 5000, 10), get(DEV, "attn", 8, 1, 5000, 10), get(DEV, "weights", 7, 1, 5000, 10)]
    held = list(CaptureScratch._held.values())  # (keeps the memory that the next capture on stream 7 lets go)
    kept.append(get(DEV, "attn", 7, 2, 5000, 10))  # another graph, captured on the same stream
    assert len(held) == 3 and len({x[0] for x in kept}) == 4
    spans = sorted((x[2], x[2] + 4 * x[3]) for x in kept)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))  # no ticket has two owners
    assert all(_bytes(x[2], 4 * x[3]) == bytes(4 * x[3]) for x in kept)
    assert get(DEV, "attn", 8, 1, 5000, 10) == kept[1]


def test_a_larger_call_keeps_what_is_large_enough():
    get = CaptureScratch.get
    small = get(DEV, "attn", 7, 1, 5000, 10)
    ctypes.memset(small[0], 0xFF, small[1])
    more_words = get(DEV, "attn", 7, 1, 300, 1000)
    assert more_words[:2] == small[:2] and more_words[3] >= 1000
    assert _bytes(more_words[2], 4 * more_words[3]) == bytes(4 * more_words[3])
    more_bytes = get(DEV, "attn", 7, 1, 9000, 10)
    assert more_bytes[2:] == more_words[2:] and more_bytes[1] >= 9000
    assert get(DEV, "attn", 7, 1, 5000, 10) == more_bytes


def test_spare_tickets_run_out():
    kept = []
    for i in range(40):
        kept.append(CaptureScratch.get(DEV, "attn", i, 1, 256, CaptureScratch.SPARE // 4 // 16))
        assert _bytes(kept[-1][2], 4 * kept[-1][3]) == bytes(4 * kept[-1][3])
        ctypes.memset(kept[-1][2], 0xFF, 4 * kept[-1][3])
    spans = sorted((x[2], x[2] + 4 * x[3]) for x in kept)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))


def test_a_null_number_is_refused():
    assert _lib.lib().mfd_capture_id(None, None) == 1
    assert b"null" in _lib.lib().mfd_last_error()
    assert _lib.lib().mfd_kv8_attention_status(None, None) != 0
