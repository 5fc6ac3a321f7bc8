"""kv8_append behind open pages whose scale no bf16 maximum gave: the codes are the stated float32 rule's, bit for bit
(test_gpu_kv8.py restates it), at the ends of the scales' range too."""
import pytest
import torch

from mfd_b200 import ops
from test_gpu_kv8 import DEV, Case, _check_append

pytestmark = pytest.mark.gpu
ONES = 2.0 - 2.0 ** -23  # a float32 significand of ones


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [2.0 ** -100, ONES * 2.0 ** -100, 1.5 * 2.0 ** -100, ONES * 2.0 ** -94, ONES * 2.0 ** -65,
                                   2.0 ** -64, ONES, 1.1, ONES * 2.0 ** 100, ONES * 2.0 ** 125, 1.3 * 2.0 ** 126, 2.0 ** 127])
def test_codes_behind_an_open_page_of_any_scale(scale, dtype):
    """Every bf16 significand at every power of two a code can tell from zero, and some beyond."""
    n = 20
    c = Case(401, [5, 16 + 9], n=n, kv=2, page=128, dtype=dtype, spare=n)
    for b in range(2):
        c.ks[int(c.table[b, 0])] = scale
        c.vs[int(c.table[b, 0])] = scale
        for codes in (c.k, c.v):  # (rows already there stay finite under every scale)
            codes[int(c.table[b, 0])] = torch.ones(codes.shape[1:], device=DEV).to(codes.dtype)
    sig = torch.arange(128, 256, device=DEV, dtype=torch.float64) / 128
    exponent = torch.arange(-13, 7, device=DEV, dtype=torch.float64)  # of x / s; below qmax for both types, nearly
    x = (sig[None, :] * torch.exp2(exponent)[:, None] * scale).clamp(max=min(100 * scale, 3e38))
    x = torch.sign(torch.randn(n, 128, device=DEV)) * x
    rows = x.bfloat16()[None, :, None].expand(2, n, 2, 128).contiguous()
    _check_append(c, rows, -rows, [list(range(n))] * 2, [n, n])
    assert c.ks[int(c.table[0, 0])].tolist() == [torch.tensor(scale, dtype=torch.float32).item()] * 2


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [2.0 ** -100, 1.0, 2.0 ** 126])
def test_zeros_of_both_signs_are_zero(scale, dtype):
    """Behind an open page, and in pages of their own, whose scale is the least."""
    c = Case(402, [5, 0], n=20, kv=2, page=16, dtype=dtype, spare=20, stale=False)
    c.ks[int(c.table[0, 0])] = scale
    rows = torch.zeros(2, 20, 2, 128, device=DEV).bfloat16()
    rows[:, ::2] = -0.0
    before = c.k[int(c.table[0, 0]), :, :5].view(torch.uint8).clone()
    lens = ops.kv8_append(c.k, c.v, c.ks, c.vs, rows, rows, c.table, c.seq)
    c.lens = lens.tolist()
    assert c.lens == [25, 20]
    assert bool((c.rows(0, "k")[:, 5:] == 0).all()) and bool((c.rows(1, "k") == 0).all()) and bool((c.rows(1, "v") == 0).all())
    assert torch.equal(c.k[int(c.table[0, 0]), :, :5].view(torch.uint8), before) and c.ks[int(c.table[0, 0])].tolist() == [scale] * 2
    assert c.ks[c.table[1, :2].long()].unique().tolist() == [2.0 ** -100]
