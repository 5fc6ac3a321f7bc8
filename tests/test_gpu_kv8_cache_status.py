"""KV8Cache after an append that found no page: its lengths count tokens that are nowhere, so it gives out and takes back no
page until its owner has looked at it."""
import pytest
import torch

from mfd_b200.kv8_cache import KV8Cache

pytestmark = pytest.mark.gpu


def _overfilled():
    cache = KV8Cache(2, 8, 1, 8, 16)
    rows = torch.randn(2, 80, 1, 128, device="cuda").bfloat16()
    cache.reserve(16)
    cache.append(rows, rows)  # 80 rows, 16 places
    return cache


def test_no_page_that_does_not_exist_becomes_free():
    cache = _overfilled()
    before = sorted(cache._free)
    with pytest.raises(RuntimeError, match="found no page"):
        cache.evict(3, sink_pages=0, recent_pages=1)
    assert sorted(cache._free) == before and all(p >= 0 for p in cache._free)


def test_no_page_is_given_to_tokens_that_were_dropped():
    cache = _overfilled()
    with pytest.raises(RuntimeError, match="found no page"):
        cache.reserve(1)
    assert cache._pages == [1, 1]
    cache.seq_lens.fill_(16)  # what the pages hold
    cache.status.zero_()
    cache.reserve(1)
    assert cache._pages == [2, 2]
