"""The 8-bit cache attention where scales and scores leave their usual ranges, in both kernels (up to 16 rows of a KV head,
and more).  References and tolerances are those of test_gpu_kv8.py, whose terms hold here too: the scores are sums of 128
float32 products, and an output is compared in units of sum p |v|, which scales with the values."""
import pytest
import torch

from mfd_b200 import ops
from test_gpu_kv8 import DEV, Case

pytestmark = pytest.mark.gpu
ROWS = [1, 4, 5, 9, 40, 65]  # nodes, of 4 heads to a KV head: the last row counts of one kernel and the first of the other


def _last_pages(c):
    return [int(c.table[b, (t - 1) // c.page]) for b, t in enumerate(c.lens) if t]


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("n", ROWS)
def test_key_scales_of_zero_in_partial_pages(n, dtype):
    """A page of zero keys may have the scale 0: its tokens score 0, and what lies behind the length stays hidden."""
    c = Case(101 + n, [0, 5, 33, 64, 290], n=n, heads=8, kv=2, page=32, dtype=dtype)
    c.ks[_last_pages(c), 0] = 0.0
    c.ks[int(c.table[4, 2])] = 0.0
    c.check()
    c.check(own=False)


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.0, -128 ** -0.5, -1.0])
def test_scales_of_zero_and_below(n, scale):
    """Softmax scales that are not positive; with -1 the scores reach 130 to either side (log2), which no float32 weight spans
    unless the reference is their maximum."""
    c = Case(111 + n, [0, 7, 150, 333], n=n, heads=8, kv=2, page=16, dtype="int8")
    c.scale = scale
    biggest = max(float((c.v.float() * c.vs[:, :, None, None]).nan_to_num().abs().max()), float(c.vn.float().abs().max()))
    for anc in (True, False):
        out, lse = c.run(anc=anc)
        ref, rl, size = c.attention(anc=anc)
        # (weights below 2^-37 of a row's largest may be lost in the kernel for few rows, as it states)
        assert bool(((out.double() - ref).abs() <= 1.05 * 2 ** -8 * size + 2.0 ** -36 * biggest).all())
        live = torch.isfinite(rl)
        assert torch.equal(lse.double()[~live], rl[~live])
        assert float(((lse.double() - rl).abs() - 2e-6 * rl.abs())[live].max()) <= 2e-5


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("leap", [9.0, 50.0])
def test_references_that_move_at_every_chunk_and_tile(leap, n, dtype):
    """Scores that rise by `leap` every 32 keys over three tiles: past 2^30 a chunk, the weights already written and O are
    scaled again within the step, several times; past 2^8 a tile, O alone at its start.  (A value read back before its store had
    finished would be a raw score, or a stale O.)"""
    c = Case(141 + n, [384, 384, 300, 130], n=n, heads=8, kv=2, page=16, dtype=dtype, stale=False)
    c.k = torch.zeros(c.k.shape, device=DEV).to(c.k.dtype)
    c.k[..., 0] = torch.full(c.k.shape[:3], 64.0, device=DEV).to(c.k.dtype)
    c.q.zero_()
    c.q[..., 0] = 1.0
    c.scale = 1.0
    for b, t in enumerate(c.lens):
        for i in range(-(-t // 16)):
            c.ks[int(c.table[b, i])] = (i // 2) * leap / 64.0
    c.check(own=False)
    c.check()


@pytest.mark.parametrize("n", [1, 9])
@pytest.mark.parametrize("codes", [0, 1])
def test_long_caches_of_zero_values(n, codes):
    """kv8_append gives a page of zeros the scale 2^-100; 70000 such tokens of one score sum to 70000 in the log-sum-exp.
    The page weights that follow from it sum to the number of rows."""
    c = Case(121, [70000, 50], n=n, heads=4, kv=1, page=128, dtype="int8", stale=False)
    c.v.fill_(codes)
    c.vs.fill_(2.0 ** -100)
    c.q.zero_()
    _, lse = c.check(own=False)
    w = ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, torch.zeros(c.table.shape, device=DEV))
    assert float((w.sum(1) - 4 * n).abs().max()) <= 4 * n * 5e-5
    c.check()


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("n", ROWS)
def test_scores_that_leap_inside_a_tile_over_values_of_any_scale(n, dtype):
    """The first page scores 0, the others 35 (50 in log2), under value scales at the floor, far above one, and mixed."""
    for vs in ((2.0 ** -100, 2.0 ** -100), (2.0 ** 100, 2.0 ** 100), (2.0 ** -100, 1.0), (1.0, 2.0 ** -100),
               (2.0 ** -50, 2.0 ** 30)):
        c = Case(131 + n, [300, 40, 31], n=n, heads=8, kv=2, page=32, dtype=dtype, stale=False)
        c.k = torch.zeros(c.k.shape, device=DEV).to(c.k.dtype)
        c.k[..., 0] = torch.full(c.k.shape[:3], 100.0 if dtype == "int8" else 96.0, device=DEV).to(c.k.dtype)
        c.q.zero_()
        c.q[..., 0] = 1.0
        c.scale = 1.0
        c.vs.fill_(vs[0])
        for b in range(3):
            ids = c.table[b, :10]
            c.ks[ids[ids >= 0].long()] = 0.35
            c.ks[int(c.table[b, 0])] = 0.0
            c.vs[ids[1::2][ids[1::2] >= 0].long()] = vs[1]
        c.check(own=False)
        c.vn *= vs[0]
        c.kn[..., 0] = 0
        c.check()
