"""KV8Cache's page bookkeeping, which is host code: a refused reservation leaves the cache as it was (no GPU)."""
import pytest
import torch

from mfd_b200.kv8_cache import KV8Cache


def _state(cache):
    return list(cache._free), list(cache._pages), cache.page_table.tolist()


def _consistent(cache):
    owned = [p for row, n in zip(cache.page_table.tolist(), cache._pages) for p in row[:n]]
    assert all(p >= 0 for p in owned) and len(set(owned)) == len(owned)
    assert sorted(owned + cache._free) == list(range(cache.k.shape[0]))


@pytest.mark.parametrize("lens,tokens,match", [
    ((0, 0), 48, "free page"),      # request 0's three pages are there, request 1's are not
    ((0, 40), 30, "table"),         # the second request is the one whose table is too narrow
    ((16, 0), 33, "free page"),
    ((0, 0), 65, "table"),
])
def test_a_refused_reservation_changes_nothing(lens, tokens, match):
    cache = KV8Cache(2, 5, 1, 4, 16, device="cpu")
    cache.reserve(16)
    cache.seq_lens = torch.tensor(lens, dtype=torch.int32)
    before = _state(cache)
    with pytest.raises(RuntimeError, match=match):
        cache.reserve(tokens)
    assert _state(cache) == before
    _consistent(cache)


def test_a_reservation_after_a_refused_one_gives_every_page_it_promises():
    cache = KV8Cache(2, 5, 1, 4, 16, device="cpu")
    with pytest.raises(RuntimeError, match="free page"):
        cache.reserve(48)
    cache._free.append(5)  # a page comes back: now there are six
    cache.k = torch.zeros(6, 1, 16, 128, dtype=torch.int8)
    cache.reserve(48)
    _consistent(cache)
    assert cache._pages == [3, 3] and all(p >= 0 for row in cache.page_table.tolist() for p in row[:3])
