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
