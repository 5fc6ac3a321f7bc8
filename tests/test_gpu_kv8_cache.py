"""KV8Cache: the operators of the 8-bit cache together, as a serving loop uses them (the example), and its page
bookkeeping: no page has two owners, freed pages come back, and the cache's values are the rows that were committed."""
import importlib.util
import os

import pytest
import torch

from mfd_b200.kv8_cache import KV8Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _owners(cache):
    table = cache.page_table.tolist()
    return [row[:n] for row, n in zip(table, cache._pages)]


def _consistent(cache):
    owned = [p for row in _owners(cache) for p in row]
    assert all(p >= 0 for p in owned) and len(set(owned)) == len(owned)
    assert not set(owned) & set(cache._free) and len(owned) + len(cache._free) == cache.k.shape[0]
    for t, n in zip(cache.seq_lens.tolist(), cache._pages):
        assert t <= n * cache.page_size


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_example_runs_and_evicts(dtype):
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "kv8_long_context.py")
    spec = importlib.util.spec_from_file_location("kv8_long_context", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(dtype, steps=5, prompt=700, page=32, keep_pages=18, log=lambda *_: None)
    cache = got["cache"]
    _consistent(cache)
    assert bool(torch.isfinite(got["out"].float()).all())
    for h in got["history"]:
        assert all(1 <= c <= 9 for c in h["committed"])
        assert all(t <= 18 * 32 for t in h["tokens"])
    assert all(e > 0 for e in got["history"][0]["evicted"])  # 700 tokens are 22 pages


@pytest.mark.parametrize("dtype,step", [(torch.int8, 1 / 254), (torch.float8_e4m3fn, 1 / 16)])
def test_cache_holds_the_rows_of_its_kept_pages(dtype, step):
    """Rows are distinguishable by value, so after several evictions every kept page is checked against the rows that
    went into it: within half a code of the page's largest value (an e4m3 code: 1 / 16 of the value)."""
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = KV8Cache(2, 60, 2, 40, 16, dtype=dtype)
    rows = torch.randn(2, 400, 2, 128, generator=g, device=DEV).bfloat16()
    cache.reserve(330)
    counts = torch.tensor([330, 100], dtype=torch.int32, device=DEV)
    cache.append(rows, -rows, counts=counts)
    _consistent(cache)
    kept = [list(range(330)), list(range(100))]
    for i, keep in enumerate((15, 9, 4)):
        cache.mass = torch.rand(cache.mass.shape, generator=g, device=DEV)
        before = _owners(cache)
        gone = cache.evict(keep, sink_pages=1, recent_pages=2)
        _consistent(cache)
        for b in range(2):
            filled = -(-len(kept[b]) // 16)
            stay = [j for j in range(filled) if before[b][j] not in set(gone[b])]
            assert len(stay) == min(filled, keep)
            kept[b] = [t for j in stay for t in kept[b][16 * j:16 * j + 16]]
        assert cache.seq_lens.tolist() == [len(k) for k in kept]
    for b in range(2):
        for j in range(-(-len(kept[b]) // 16)):
            want = rows[b, kept[b][16 * j:16 * j + 16]].transpose(0, 1).float()
            page = int(cache.page_table[b, j])
            for codes, scale, sign in ((cache.k, cache.k_scale, 1), (cache.v, cache.v_scale, -1)):
                got = sign * codes[page, :, :want.shape[1]].float() * scale[page][:, None, None]
                big = want.abs().amax((1, 2), keepdim=True)
                tol = step * 1.001 * (big if dtype == torch.int8 else torch.maximum(want.abs(), big / 448))
                assert bool(((got - want).abs() <= tol).all())


def test_reserve_refuses_what_it_cannot_give():
    cache = KV8Cache(2, 5, 1, 4, 16)
    with pytest.raises(RuntimeError, match="table"):
        cache.reserve(65)
    with pytest.raises(RuntimeError, match="free page"):
        cache.reserve(48)
    cache = KV8Cache(1, 5, 1, 4, 16)
    rows = torch.zeros(1, 20, 1, 128, dtype=torch.bfloat16, device=DEV)
    cache.reserve(16)
    cache.append(rows, rows)  # 20 rows, 16 places
    assert int(cache.status) == 4
