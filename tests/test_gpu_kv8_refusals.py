"""Arguments of the 8-bit cache operators that are refused, beside those of test_gpu_kv8.py, and calls that are not."""
import pytest
import torch

from mfd_b200 import ops
from test_gpu_kv8 import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("status", [torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64),
                                    torch.zeros(0, dtype=torch.int32), torch.zeros(1)])
def test_append_refuses_a_status_that_is_no_int32(status):
    c = Case(301, [4, 30], n=6, kv=2, page=16, dtype="int8", spare=8)
    before = [t.clone() for t in (c.k, c.v)]
    with pytest.raises(RuntimeError, match="status"):
        ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn, c.vn, c.table, c.seq, status=status.to(DEV))
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])


@pytest.mark.parametrize("n", [1, 40])
def test_an_empty_batch_gives_empty_results(n):
    c = Case(302, [20, 3], n=n, heads=4, kv=2, page=16, dtype="int8")
    none = dict(k_new=c.kn[:0], v_new=c.vn[:0])
    out, lse = ops.kv8_attention(c.q[:0], c.k, c.v, c.ks, c.vs, c.table[:0], c.seq[:0], 1.0, **none, return_lse=True)
    assert out.shape == (0, n, 4, 128) and lse.shape == (0, n, 4)
    mass = torch.zeros(c.table.shape, device=DEV)[:0]
    assert ops.kv8_page_weights(c.q[:0], lse, c.k, c.ks, c.table[:0], c.seq[:0], 1.0, mass).shape == mass.shape
    assert ops.kv8_append(c.k, c.v, c.ks, c.vs, *none.values(), c.table[:0], c.seq[:0]).shape == (0,)
    assert [tuple(t.shape) for t in ops.kv8_evict(c.table[:0], mass, c.seq[:0], 16, 4, 1, 1)][2:] == [(0,), mass.shape, (0,)]


@pytest.mark.parametrize("bs,n", [(1, 1), (1, 3), (2, 1)])
def test_keys_and_values_whose_strides_differ_where_it_does_not_matter(bs, n):
    """A decode step's rotated keys are a tensor of their own, its values a slice of the fused projection: a batch of one, or
    one node, has strides that address nothing."""
    c = Case(303, [70] * bs, n=n, heads=4, kv=2, page=16, dtype="int8", spare=8)
    want = c.run()
    if bs == 1:
        c.vn = torch.cat([c.vn, c.vn], 1)[:, :n]
    else:
        c.kn, c.vn = c.kn.transpose(0, 1).contiguous().transpose(0, 1), c.vn.as_strided(c.vn.shape, (256, 9 * 256, 128, 1))
        c.kn = c.kn.as_strided(c.kn.shape, (256, 7 * 256, 128, 1))
    assert c.kn.stride() != c.vn.stride()
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn, c.vn, c.table, c.seq)


def test_keys_and_values_whose_strides_differ_where_it_matters():
    c = Case(304, [70, 3], n=2, heads=4, kv=2, page=16, dtype="int8", spare=8)
    c.vn = torch.cat([c.vn, c.vn], 1)[:, :2]
    with pytest.raises(RuntimeError, match="strides"):
        c.run()
    with pytest.raises(RuntimeError, match="strides"):
        ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn, c.vn, c.table, c.seq)
