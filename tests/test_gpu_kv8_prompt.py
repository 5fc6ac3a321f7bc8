"""The 8-bit cache attention of a prompt's chunk: many nodes that see one another up to themselves (no mask given), behind an
empty cache and behind others; rows of several blocks, and own keys of several tiles.  References and tolerances are those of
test_gpu_kv8.py."""
import pytest
import torch

from test_gpu_kv8 import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [127, 129, 256, 300, 700])
def test_a_prompt_chunk_attends_to_itself(n, dtype):
    Case(501 + n, [0, 100, 1, 640], n=n, heads=4, kv=2, page=64, dtype=dtype).check(anc=False)


@pytest.mark.parametrize("heads,kv,n", [(3, 1, 257), (1, 1, 1100), (8, 1, 130)])
def test_prompt_chunks_of_other_head_groups(heads, kv, n):
    Case(511 + n, [0, 33], n=n, heads=heads, kv=kv, page=16, dtype="int8").check(anc=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_chunk_does_not_see_does_not_reach_it(bad):
    """Every node from the 200th on is non-finite: the rows before it are as if those were not there."""
    n = 300
    c = Case(521, [0, 50], n=n, heads=4, kv=2, page=32, dtype="e4m3")
    c.kn[:, 200:], c.vn[:, 200:] = bad, bad
    out, lse = c.run(anc=False)
    c.kn[:, 200:], c.vn[:, 200:] = 0, 0
    ref, rl, size = c.attention(anc=False)
    assert float(((out.double() - ref).abs() - 1.05 * 2 ** -8 * size)[:, :200].max()) <= 1e-30
    assert float(((lse.double() - rl).abs() - 2e-6 * rl.abs())[:, :200].max()) <= 2e-5
    assert not bool(torch.isfinite(out[:, 200:].float()).any())
