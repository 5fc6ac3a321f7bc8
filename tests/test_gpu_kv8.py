"""The 8-bit paged K/V cache (append, attention, page weights, eviction) against plain implementations.

References are in float64 (attention, weights), in the stated float32 rule (append: the codes are exact) and in plain
Python (eviction: exact).  Tolerances, fixed before the first run:
  attention   |out - ref| <= 1.05 * 2^-8 * sum_j p_j |v_j|: the output's rounding to bf16 alone may take 2^-8 of |out|,
              so the weights may lose next to nothing (the kernels keep 16 bits of each)
  lse         2e-5 + 2e-6 |lse|: 128-term float32 sums of products of size up to about 15, a few of their last places
  weights     5e-5 relative (the exponential of a score error of at most 2e-5, and float32 sums)
"""
import numpy as np
import pytest
import torch

from mfd_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Case:
    """A cache with random codes, scattered pages and rows for bs requests."""

    def __init__(self, seed, lens, n=1, heads=8, kv=2, page=32, dtype="int8", spare=0, layout="phtd", stale=True):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.lens, self.n, self.heads, self.kv, self.page, self.dtype = list(lens), n, heads, kv, page, dtype
        bs = len(self.lens)
        need = [-(-(t + spare) // page) for t in self.lens]
        pool = sum(need) + 3
        ids = rng.permutation(pool)
        width = max(1, max(need)) + 2
        table = np.full((bs, width), -1, np.int32)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = ids[at:at + m]
            at += m
        self.table = torch.from_numpy(table).to(DEV)
        self.seq = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        shape = (pool, kv, page, D) if layout == "phtd" else (pool, page, kv, D)

        def codes():
            x = torch.randn(shape, generator=g, device=DEV)
            c = (x * 36).round().clamp(-127, 127).to(torch.int8) if dtype == "int8" else (x * 128).clamp(-448, 448).to(
                torch.float8_e4m3fn)
            return c if layout == "phtd" else c.transpose(1, 2)

        self.k, self.v = codes(), codes()
        q = 127.0 if dtype == "int8" else 448.0
        self.ks = torch.exp(torch.randn(pool, kv, generator=g, device=DEV) * 0.5) * 3.5 / q
        self.vs = torch.exp(torch.randn(pool, kv, generator=g, device=DEV) * 1.5) * 3.5 / q
        if stale:  # whatever is behind the length must not matter: NaN codes (e4m3), NaN scales of unused pages
            used = torch.zeros(pool, dtype=torch.bool)
            for b, t in enumerate(self.lens):
                for p in range(-(-t // page)):
                    used[int(table[b, p])] = True
                if t % page:
                    last = int(table[b, t // page])
                    for c in (self.k, self.v):
                        c[last, :, t % page:] = float("nan") if dtype == "e4m3" else -128
            for c in (self.k, self.v):
                c.view(torch.uint8)[~used.to(DEV)] = 0x7F
            self.ks[~used.to(DEV)] = float("nan")
            self.vs[~used.to(DEV)] = float("nan")
        self.q = (torch.randn(bs, n, heads, D, generator=g, device=DEV) * 2).bfloat16()
        self.kn = torch.randn(bs, n, kv, D, generator=g, device=DEV).bfloat16()
        self.vn = torch.randn(bs, n, kv, D, generator=g, device=DEV).bfloat16()
        sets = []
        for _ in range(bs):
            one = [1]
            for i in range(1, n):
                one.append(one[int(rng.integers(max(0, i - 6), i))] | (1 << i))
            sets.append(one)
        self.sets = sets
        self.scale = D ** -0.5

    def anc(self, extra_words=0):
        words = (self.n + 63) // 64 + extra_words
        w = np.array([[[(s >> (64 * j)) & (2 ** 64 - 1) for j in range(words)] for s in one] for one in self.sets],
                     dtype=np.uint64)
        return torch.from_numpy(w.view(np.int64)).to(DEV)

    def visible(self, b):
        return torch.tensor([[(s >> j) & 1 for j in range(self.n)] for s in self.sets[b]], dtype=torch.bool, device=DEV)

    def rows(self, b, name):
        c, s = (self.k, self.ks) if name == "k" else (self.v, self.vs)
        t = self.lens[b]
        ids = self.table[b, :-(-t // self.page)].long()
        x = c.contiguous().view(torch.uint8)[ids].view(c.dtype).double() * s[ids].double()[:, :, None, None]
        return x.transpose(0, 1).reshape(self.kv, -1, D)[:, :t]

    def attention(self, own=True, anc=True):
        """(out, lse, sum p |v|) in float64."""
        bs, g = len(self.lens), self.heads // self.kv
        out = torch.zeros(bs, self.n, self.heads, D, dtype=torch.float64, device=DEV)
        size, lse = torch.zeros_like(out), torch.zeros(bs, self.n, self.heads, dtype=torch.float64, device=DEV)
        for b in range(bs):
            t = self.lens[b]
            k, v = self.rows(b, "k"), self.rows(b, "v")
            if own:
                k = torch.cat([k, self.kn[b].double().transpose(0, 1)], 1)
                v = torch.cat([v, self.vn[b].double().transpose(0, 1)], 1)
                see = self.visible(b) if anc else torch.tril(torch.ones(self.n, self.n, dtype=torch.bool, device=DEV))
                see = torch.cat([torch.ones(self.n, t, dtype=torch.bool, device=DEV), see], 1)
            else:
                see = torch.ones(self.n, t, dtype=torch.bool, device=DEV)
            for h in range(self.heads):
                s = self.q[b, :, h].double() @ k[h // g].T * self.scale
                s = torch.where(see, s, torch.full_like(s, -float("inf")))
                l = torch.logsumexp(s, 1) if s.shape[1] else torch.full((self.n,), -float("inf"), device=DEV).double()
                p = torch.where(see, torch.exp(s - l[:, None]), torch.zeros_like(s))
                p = torch.where(torch.isneginf(l)[:, None], torch.zeros_like(p), p)
                for i in range(self.n):  # a row's sum runs over what it sees, so a value it does not see is not there
                    if s.shape[1] and not bool(torch.isfinite(v[h // g]).all()):
                        out[b, i, h] = p[i][see[i]] @ v[h // g][see[i]]
                if bool(torch.isfinite(v[h // g]).all()):
                    out[b, :, h] = p @ v[h // g]
                size[b, :, h] = p @ torch.nan_to_num(v[h // g].abs(), posinf=0.0)
                lse[b, :, h] = l
        return out, lse, size

    def run(self, own=True, anc=True, **kw):
        return ops.kv8_attention(self.q, self.k, self.v, self.ks, self.vs, self.table, self.seq, self.scale,
                                 k_new=self.kn if own else None, v_new=self.vn if own else None,
                                 anc=self.anc() if own and anc else None, return_lse=True, **kw)

    def check(self, own=True, anc=True, got=None):
        out, lse = got if got is not None else self.run(own, anc)
        ref, rl, size = self.attention(own, anc)
        assert out.dtype == torch.bfloat16 and lse.dtype == torch.float32
        fine = torch.isfinite(ref)
        x = out.double()
        assert torch.equal(torch.isnan(x), torch.isnan(ref)) and torch.equal(x[torch.isinf(ref)], ref[torch.isinf(ref)])
        err = ((x - ref).abs() - 1.05 * 2 ** -8 * size)[fine]
        assert err.numel() == 0 or float(err.max()) <= 1e-30, float(err.max())
        live = torch.isfinite(rl)
        assert torch.equal(lse.double()[~live], rl[~live])
        el = ((lse.double() - rl).abs() - 2e-6 * rl.abs())[live]
        assert el.numel() == 0 or float(el.max()) <= 2e-5, float(el.max())
        assert ops.kv8_attention_status() == 0
        return out, lse


# ------------------------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 17, 65])
def test_attention_lengths_pages_and_types(dtype, page, n):
    """Lengths around groups, pages and tiles, empty and one-token requests among them."""
    lens = [0, 1, 15, 16, 17, page - 1, page, page + 1, 127, 128, 129, 300, 1000]
    Case(n * 1000 + page, lens, n=n, heads=8, kv=2, page=page, dtype=dtype).check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (7, 1), (8, 1), (16, 1), (20, 4), (28, 4), (40, 8), (64, 2)])
@pytest.mark.parametrize("n", [1, 4, 33])
def test_attention_head_groups(heads, kv, n):
    """Group sizes from 1 to 32, odd ones among them, for decode, a short draft and a small tree."""
    Case(heads * 100 + n, [5, 190, 0, 64], n=n, heads=heads, kv=kv, page=16, dtype="e4m3").check()


@pytest.mark.parametrize("n", [64, 65, 128, 129, 200, 513])
def test_attention_large_trees(n):
    """Mask words, row tiles and own-key tiles that end inside and on their boundaries."""
    Case(n, [0, 260, 1], n=n, heads=4, kv=2, page=64, dtype="int8").check()


@pytest.mark.parametrize("n", [1, 6, 65])
def test_attention_without_own_keys_and_without_a_mask(n):
    c = Case(7 + n, [0, 1, 77, 512], n=n, heads=8, kv=2, page=32, dtype="e4m3")
    c.check(own=False)  # (a row that sees nothing: 0 and -inf)
    c.check(anc=False)  # a chain


@pytest.mark.parametrize("n", [3, 40, 100])
def test_attention_rows_whose_mask_is_empty(n):
    """Padding nodes with no bit set, behind an empty and a non-empty cache."""
    c = Case(11, [0, 50], n=n, heads=4, kv=2, page=16, dtype="int8")
    for one in c.sets:
        for i in range(1, n, 2):
            one[i] = 0
    out, lse = c.check()
    assert bool((out[0, 1] == 0).all()) and bool(torch.isneginf(lse[0, 1]).all())


@pytest.mark.parametrize("n", [3, 24, 80])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_non_finite_own_keys_stay_where_they_are_seen(n, bad):
    """A node's non-finite key or value reaches the rows that see the node and no other row."""
    c = Case(13 + n, [0, 33, 150], n=n, heads=4, kv=2, page=16, dtype="e4m3")
    i = n // 2
    c.vn[1, i, 0, 5] = bad
    c.vn[1, i, 1, 127] = bad
    c.check()
    c = Case(14 + n, [20, 33], n=n, heads=4, kv=2, page=16, dtype="int8")
    for one in c.sets:  # nobody but itself sees the last node
        one[n - 1] = 1 << (n - 1)
    c.kn[1, n - 1] = bad
    c.vn[1, n - 1] = bad
    out, _ = c.run()
    ref, _, size = c.attention()
    assert bool(torch.isfinite(out[:, :n - 1].float()).all())
    assert float(((out.double() - ref).abs() - 1.05 * 2 ** -8 * size)[:, :n - 1].max()) <= 1e-30


@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_layouts_and_strides(n):
    """Token-major pages, queries and keys sliced out of a fused projection, a strided output, a wide table."""
    c = Case(17, [100, 3, 0, 259], n=n, heads=6, kv=2, page=32, dtype="int8", layout="pthd")
    bs = 4
    fused = torch.randn(bs, n, 6 + 2 + 2, D, device=DEV).bfloat16()
    c.q, c.kn, c.vn = fused[:, :, :6], fused[:, :, 6:8], fused[:, :, 8:]
    wide = torch.full((bs, n, 9, D), 7.0, dtype=torch.bfloat16, device=DEV)
    big = torch.full((bs, 50), -1, dtype=torch.int32, device=DEV)
    big[:, 3:3 + c.table.shape[1]] = c.table
    c.table = big[:, 3:]
    got = c.run(out=wide[:, :, 1:7])
    c.check(got=got)
    assert bool((wide[:, :, 0] == 7).all()) and bool((wide[:, :, 7:] == 7).all())


@pytest.mark.parametrize("n", [1, 9, 65])
@pytest.mark.parametrize("bs", [40, 300])
def test_attention_many_requests(bs, n):
    """More requests than a warp has lanes, lengths from 0 up, several units per CTA."""
    rng = np.random.default_rng(bs)
    Case(bs, rng.integers(0, 90, bs).tolist(), n=n, heads=4, kv=1, page=16, dtype="e4m3").check()


@pytest.mark.parametrize("n", [1, 3, 20, 65])
def test_attention_many_units_of_very_unequal_lengths(n):
    # more units than half the CTAs of either kernel, so CTAs' ranges begin and end inside units, and in what a unit is
    # counted for beside its tiles
    Case(23 + n, [3000, 0, 1, 2, 0, 129, 16, 0, 1700, 5, 0, 0, 127, 128, 1, 640] * 3, n=n, heads=16, kv=4, page=16).check()


@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("tokens", [129, 4096, 40000])
def test_attention_one_request_in_many_pieces(n, tokens):
    Case(29 + n, [tokens], n=n, heads=4, kv=1, page=64).check()


@pytest.mark.parametrize("n", [1, 12, 65])
def test_attention_long_requests_are_split_and_merged(n):
    """One long request over the whole GPU, next to short ones; and the same bits every time."""
    c = Case(19, [40003], n=n, heads=4, kv=1, page=64, dtype="int8")
    a = c.check()
    for _ in range(3):
        b = c.run()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    Case(20, [20000, 3, 0, 777], n=n, heads=8, kv=2, page=128, dtype="e4m3").check()


@pytest.mark.parametrize("n", [1, 30])
def test_attention_score_ranges(n):
    """Scores that rise along the cache (the running maximum moves), large queries, a zero query row."""
    c = Case(23, [600], n=n, heads=4, kv=1, page=32, dtype="int8", stale=False)
    ids = c.table[0, :19].long()
    c.ks[ids] = (torch.arange(1, 20, device=DEV) * 0.02)[:, None]
    c.q *= 4
    c.q[0, 0, 1] = 0
    c.check()
    c = Case(24, [90], n=n, heads=4, kv=1, page=16, dtype="e4m3", stale=False)
    c.q = (c.q.float() * 2.0 ** 100).bfloat16()  # far outside float16; the scale brings the scores back
    c.scale *= 2.0 ** -100
    c.check()
    c.q = (c.q.float() * 2.0 ** -200).bfloat16()
    c.scale *= 2.0 ** 200
    c.vs *= 2.0 ** -60
    c.vn *= 0
    out, _ = c.run()
    ref, _, size = c.attention()
    assert float(((out.double() - ref).abs() - 1.05 * 2 ** -8 * size).max()) <= 2.0 ** -126


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 codes whose last pages are in use."""
    page, kv = 128, 8
    pool = (1 << 32) // (page * kv * D) + 40
    c = Case(29, [500, 129], n=2, heads=16, kv=kv, page=page, dtype="int8", stale=False)
    small = c.k.shape[0]
    for name in ("k", "v"):
        big = torch.empty(pool, kv, page, D, dtype=torch.int8, device=DEV)
        big[-small:] = getattr(c, name)
        setattr(c, name, big)
        s = torch.ones(pool, kv, device=DEV)
        s[-small:] = getattr(c, name + "s")
        setattr(c, name + "s", s)
    c.table = torch.where(c.table >= 0, c.table + (pool - small), c.table)
    got = c.run()
    c.k, c.v, c.ks, c.vs = c.k[-small:], c.v[-small:], c.ks[-small:].contiguous(), c.vs[-small:].contiguous()
    c.table = torch.where(c.table >= 0, c.table - (pool - small), c.table)
    c.check(got=got)


def test_attention_bad_table_entries_read_inside_the_pool():
    """Ids outside the pool are clamped: whatever comes out, the other requests are right and nothing faults."""
    c = Case(31, [100, 100], n=2, heads=4, kv=2, page=16, dtype="int8", stale=False)
    bad = c.table.clone()
    bad[0, 0], bad[0, 1] = 2 ** 31 - 1, -5
    good, table = c.run(), c.table
    c.table = bad
    got = c.run()
    c.table = table
    assert torch.equal(good[0][1], got[0][1]) and torch.equal(good[1][1], got[1][1])


@pytest.mark.parametrize("n", [1, 40])
def test_attention_graph_replay_with_new_lengths_and_on_two_streams(n):
    c = Case(37, [700, 64, 0, 333], n=n, heads=8, kv=2, page=32, dtype="int8", stale=False)
    anc = c.anc()
    args = (c.q, c.k, c.v, c.ks, c.vs, c.table, c.seq, c.scale)
    kw = dict(k_new=c.kn, v_new=c.vn, anc=anc, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv8_attention(*args, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.kv8_attention(*args, **kw)
    for lens in ([700, 64, 0, 333], [3, 20, 0, 1], [699, 1, 0, 300]):
        c.lens = lens
        c.seq.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c.check(got=got)
    # two streams at once, each with its own scratch
    want = ops.kv8_attention(*args, **kw)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [ops.kv8_attention(*args, **kw) for _ in range(20)]
    torch.cuda.synchronize()
    for out, lse in outs:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ---------------------------------------------------------------------------------------------------------- append

def _encode(x, dtype):
    if dtype == "int8":
        return x.clamp(-127, 127).round().to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(c, kn, vn, path, counts):
    """The stated rule, one page at a time, in float32."""
    qmax = 127.0 if c.dtype == "int8" else 448.0
    out = []
    for codes, scales, new in ((c.k.clone(), c.ks.clone(), kn), (c.v.clone(), c.vs.clone(), vn)):
        for b, t in enumerate(c.lens):
            for h in range(c.kv):
                i = 0
                while i < counts[b]:
                    slot = (t + i) % c.page
                    m = min(c.page - slot, counts[b] - i)
                    p = int(c.table[b, (t + i) // c.page])
                    x = torch.stack([new[b, path[b][i + j], h].float() for j in range(m)])
                    fin = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
                    s = torch.maximum(fin.amax() * torch.tensor(1 / qmax, device=DEV), torch.tensor(2.0 ** -100, device=DEV))
                    if slot:
                        old = scales[p, h].clone()
                        s = torch.maximum(s, old)
                        keep = codes[p, h, :slot].float() * old
                        codes[p, h, :slot] = _encode(keep / s, c.dtype)
                    y = torch.nan_to_num(x / s, nan=0.0, posinf=qmax, neginf=-qmax)
                    codes[p, h, slot:slot + m] = _encode(y, c.dtype)
                    scales[p, h] = s
                    i += m
        out += [codes, scales]
    return out


def _check_append(c, kn, vn, nodes, rows, **kw):
    want = _plain_append(c, kn, vn, nodes, rows)
    lens = ops.kv8_append(c.k, c.v, c.ks, c.vs, kn, vn, c.table, c.seq, **kw)
    assert lens.tolist() == [t + m for t, m in zip(c.lens, rows)]
    for got, ref in zip((c.k, c.ks, c.v, c.vs), want):
        if got.dtype in DTYPES.values():
            got, ref = got.contiguous().view(torch.uint8), ref.contiguous().view(torch.uint8)
        else:
            got, ref = got.view(torch.int32), ref.view(torch.int32)  # (unused pages' scales are NaN)
        assert torch.equal(got, ref)
    return lens


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["phtd", "pthd"])
def test_append_paths(dtype, page, layout):
    """Accepted paths behind open, full and empty pages; rows that raise a page's scale and rows that do not."""
    lens = [0, 1, page - 1, page, page + 1, 3 * page - 5]
    c = Case(page, lens, n=30, kv=2, page=page, dtype=dtype, spare=20, layout=layout)
    counts = [1, 17, 5, 16, 0, 17]
    rng = np.random.default_rng(3)
    path = [sorted(rng.choice(30, m, replace=False).tolist()) for m in counts]
    t = torch.tensor([p + [-1] * (17 - len(p)) for p in path], dtype=torch.int64, device=DEV)
    kn, vn = c.kn.clone(), c.vn.clone()
    kn[2] *= 20
    vn[3] *= 0.01
    kn[1, :, :, 7] = 0
    vn[5] = 0
    _check_append(c, kn, vn, path, counts, path=t)
    assert bool(torch.isfinite(c.ks[c.table[5, 0].long()]).all())


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_append_counts_prompts_and_strided_rows(dtype):
    lens, counts = [0, 77, 128], [300, 0, 129]
    c = Case(41, lens, n=300, kv=3, page=64, dtype=dtype, spare=300)
    fused = torch.randn(3, 300, 7, D, device=DEV).bfloat16()
    _check_append(c, fused[:, :, 1:4], fused[:, :, 4:], [list(range(300))] * 3, counts,
                  counts=torch.tensor(counts, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_append_non_finite_and_tiny_values(dtype):
    c = Case(43, [5, 0], n=4, kv=2, page=16, dtype=dtype, spare=8)
    kn, vn = c.kn.clone(), c.vn.clone()
    kn[0, 1, 0, 3], kn[0, 1, 1, 4], kn[1, 2, 0, 9] = float("inf"), -float("inf"), float("nan")
    vn[1] = float("nan")
    vn[0] *= 2.0 ** -120
    _check_append(c, kn, vn, [list(range(4))] * 2, [4, 4])
    assert float(c.vs[int(c.table[1, 0]), 0]) == 2.0 ** -100


def test_append_stops_at_invalid_nodes_and_at_the_capacity():
    c = Case(47, [4, 30, 0], n=6, kv=2, page=16, dtype="int8", spare=8)
    c.table = c.table[:, :2].contiguous()  # 32 tokens a request
    path = torch.tensor([[0, 3, 9, 1], [0, 1, 2, 3], [0, 2, 4, 5]], dtype=torch.int64, device=DEV)
    c.table[2, 0] = 10 ** 6
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    k0 = c.k.clone()
    want = _plain_append(c, c.kn, c.vn, [[0, 3], [0, 1], []], [2, 2, 0])
    lens = ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn, c.vn, c.table, c.seq, path=path, status=status)
    assert lens.tolist() == [6, 32, 4] and int(status) == 4
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[2]) and not torch.equal(c.k, k0)


def test_append_in_steps_equals_the_values_it_was_given():
    """Token by token the scale only grows and a row is rounded again at most when it does: the error stays below
    half a step of the final scale for each growth."""
    for dtype, step in (("int8", 1.0), ("e4m3", 32.0)):
        c = Case(53, [0], n=40, kv=2, page=16, dtype=dtype, spare=40, stale=False)
        lens = c.seq
        for i in range(40):
            lens = ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn[:, i:i + 1], c.vn[:, i:i + 1], c.table, lens)
        assert int(lens) == 40
        c.lens = [40]
        for name, new, s in (("k", c.kn, c.ks), ("v", c.vn, c.vs)):
            got = c.rows(0, name)
            ref = new[0].double().transpose(0, 1)
            big = s[c.table[0, :3].long()].max().double()
            assert float((got - ref).abs().max()) <= float(big) * step * 0.5 * 8


# --------------------------------------------------------------------------------------------------------- weights

def _check_weights(c, nodes, rows, decay, **kw):
    _, lse = c.run()
    mass = torch.rand(c.table.shape, device=DEV)
    got = ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, mass, decay=decay, **kw)
    g = c.heads // c.kv
    ref = torch.zeros(c.table.shape, dtype=torch.float64, device=DEV)
    for b, t in enumerate(c.lens):
        pages = -(-t // c.page)
        w = torch.zeros(pages * c.page, dtype=torch.float64, device=DEV)
        k = c.rows(b, "k")
        for h in range(c.heads):
            for i in nodes[b][:rows[b]]:
                w[:t] += torch.exp(k[h // g] @ c.q[b, i, h].double() * c.scale - lse[b, i, h].double())
        ref[b, :pages] = mass[b, :pages].double() * decay + w.view(pages, c.page).sum(1)
    assert bool((got[ref == 0] == 0).all())
    assert float(((got.double() - ref).abs() / ref.clamp_min(1e-30)).max()) <= 5e-5
    again = ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, mass, decay=decay, out=mass, **kw)
    assert again.data_ptr() == mass.data_ptr() and torch.equal(again, got)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(8, 2), (7, 1), (32, 8)])
def test_weights_of_accepted_paths(dtype, page, heads, kv):
    lens = [0, 1, 17, page, 3 * page + 5, 700]
    c = Case(page + heads, lens, n=20, heads=heads, kv=kv, page=page, dtype=dtype)
    counts = [2, 1, 17, 4, 0, 9]
    rng = np.random.default_rng(5)
    path = [sorted(rng.choice(20, m, replace=False).tolist()) for m in counts]
    t = torch.tensor([p + [-1] * (17 - len(p)) for p in path], dtype=torch.int64, device=DEV)
    _check_weights(c, path, counts, 0.75, path=t)


def test_weights_of_counted_rows_many_rows_and_many_requests():
    counts = [65, 0, 30]
    c = Case(59, [500, 20, 64], n=65, heads=16, kv=2, page=32, dtype="int8")  # 520 rows a KV head: staged in parts
    _check_weights(c, [list(range(65))] * 3, counts, 1.0, counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
    rng = np.random.default_rng(6)
    c = Case(60, rng.integers(0, 100, 70).tolist(), n=3, heads=4, kv=2, page=16, dtype="e4m3")
    _check_weights(c, [[0, 1, 2]] * 70, [3] * 70, 0.0)
    c = Case(61, [30000], n=3, heads=4, kv=1, page=128, dtype="int8")
    _check_weights(c, [[0, 1, 2]], [3], 0.5)


def test_weights_of_a_row_that_saw_nothing_are_zero():
    c = Case(67, [64], n=2, heads=2, kv=1, page=16, dtype="int8")
    lse = torch.full((1, 2, 2), -float("inf"), device=DEV)
    mass = torch.ones(c.table.shape, device=DEV)
    got = ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, mass)
    assert got[0, :4].tolist() == [1.0] * 4 and bool((got[0, 4:] == 0).all())


# -------------------------------------------------------------------------------------------------------- eviction

def _plain_evict(table, mass, lens, page, keep, sink, recent):
    t2, m2, l2, f2, c2 = [], [], [], [], []
    width = len(table[0])
    for row, ms, t in zip(table, mass, lens):
        pages = -(-t // page)
        stay = list(range(pages))
        if pages > keep:
            middle = list(range(sink, pages - recent))
            key = lambda i: (-ms[i] if ms[i] == ms[i] else float("inf"), i)  # noqa: E731
            won = set(sorted(middle, key=key)[:keep - sink - recent])
            stay = [i for i in range(pages) if i < sink or i >= pages - recent or i in won]
        gone = [i for i in range(pages) if i not in set(stay)]
        t2.append([row[i] for i in stay] + [-1] * (width - len(stay)))
        m2.append([ms[i] for i in stay] + [0.0] * (width - len(stay)))
        f2.append([row[i] for i in gone] + [-1] * (width - len(gone)))
        l2.append(t - len(gone) * page)
        c2.append(len(gone))
    return t2, m2, l2, f2, c2


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("width,keep,sink,recent", [(1, 1, 0, 1), (8, 3, 1, 1), (40, 40, 2, 4), (100, 33, 0, 32),
                                                    (100, 33, 1, 32), (1024, 700, 4, 16), (1030, 6, 4, 1),
                                                    (3000, 2999, 0, 1), (40000, 12345, 3, 9)])
def test_eviction(page, width, keep, sink, recent):
    """Budgets of every kind, lengths under and over them, equal masses, zeros of both signs, infinities and NaN."""
    rng = np.random.default_rng(width + page)
    lens = [width * page, max(0, width * page - 3), width * page // 2, 0, min(width, keep) * page, min(width, keep + 1) * page - 1]
    bs = len(lens)
    mass = rng.exponential(size=(bs, width)).astype(np.float32) ** 4
    mass[0] = np.round(mass[0])
    mass[1, ::3] = 0.0
    mass[1, 1::6] = -0.0
    mass[2] = 1.5
    mass[5, rng.integers(0, width, max(1, width // 50))] = np.nan
    mass[5, rng.integers(0, width, max(1, width // 50))] = np.inf
    table = rng.integers(0, 2 ** 31 - 1, (bs, width), dtype=np.int64).astype(np.int32)
    got = ops.kv8_evict(torch.from_numpy(table).to(DEV), torch.from_numpy(mass).to(DEV),
                        torch.tensor(lens, dtype=torch.int32, device=DEV), page, keep, sink, recent)
    want = _plain_evict(table.tolist(), mass.tolist(), lens, page, keep, sink, recent)
    assert got[0].tolist() == want[0] and got[2].tolist() == want[2]
    assert got[3].tolist() == want[3] and got[4].tolist() == want[4]
    np.testing.assert_array_equal(got[1].cpu().numpy(), np.array(want[1], np.float32))


# -------------------------------------------------------------------------------------------------------- refusals

def test_refusals():
    c = Case(71, [20], n=2, heads=4, kv=2, page=16, dtype="int8")
    att = lambda **kw: ops.kv8_attention(**{**dict(q=c.q, k_cache=c.k, v_cache=c.v, k_scale=c.ks, v_scale=c.vs,  # noqa: E731
                                                   page_table=c.table, seq_lens=c.seq, scale=1.0, k_new=c.kn,
                                                   v_new=c.vn, anc=c.anc()), **kw})
    att()
    for kw in (dict(q=c.q.float()), dict(q=c.q[:, :, :3]), dict(q=c.q.transpose(2, 3)), dict(k_cache=c.k.half()),
               dict(v_cache=c.v[:, :, :8]), dict(k_scale=c.ks.double()), dict(v_scale=c.vs[:1]),
               dict(page_table=c.table.long()), dict(seq_lens=c.seq.long()), dict(seq_lens=c.seq.repeat(2)),
               dict(k_new=None), dict(k_new=c.kn[:, :1]), dict(v_new=c.vn.repeat(1, 1, 2, 1)[:, :, ::2]),
               dict(anc=c.anc().int()), dict(anc=c.anc()[:, :1]), dict(page_table=c.table.cpu()),
               dict(k_cache=c.k[..., :64], v_cache=c.v[..., :64], q=c.q[..., :64], k_new=None, v_new=None)):
        with pytest.raises(RuntimeError):
            att(**kw)
    wide = torch.zeros(1, 70, 4, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="mask words"):
        att(q=wide, k_new=wide[:, :, :2], v_new=wide[:, :, 2:], anc=torch.zeros(1, 70, 1, dtype=torch.int64, device=DEV))
    odd = torch.zeros(4 * 2 * 24 * D, dtype=torch.int8, device=DEV).view(4, 2, 24, D)
    with pytest.raises(RuntimeError, match="page size"):
        att(k_cache=odd, v_cache=odd, k_scale=torch.ones(4, 2, device=DEV), v_scale=torch.ones(4, 2, device=DEV))
    app = lambda **kw: ops.kv8_append(**{**dict(k_cache=c.k, v_cache=c.v, k_scale=c.ks, v_scale=c.vs, k_new=c.kn,  # noqa: E731
                                                v_new=c.vn, page_table=c.table, seq_lens=c.seq), **kw})
    path = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    for kw in (dict(path=path.int()), dict(path=path.repeat(2, 1)), dict(counts=torch.ones(1, device=DEV)),
               dict(new_lens=c.seq), dict(new_lens=c.seq.long()), dict(k_new=c.kn.float()), dict(k_new=c.kn[:, :, :1])):
        with pytest.raises(RuntimeError):
            app(**kw)
    lse = torch.zeros(1, 2, 4, device=DEV)
    mass = torch.zeros(c.table.shape, device=DEV)
    wei = lambda **kw: ops.kv8_page_weights(**{**dict(q=c.q, lse=lse, k_cache=c.k, k_scale=c.ks, page_table=c.table,  # noqa: E731
                                                      seq_lens=c.seq, scale=1.0, mass=mass), **kw})
    for kw in (dict(lse=lse.double()), dict(lse=lse[:, :1]), dict(mass=mass[:, :1]), dict(mass=mass.half()),
               dict(out=mass.double()), dict(path=path.int())):
        with pytest.raises(RuntimeError):
            wei(**kw)
    evi = lambda *a: ops.kv8_evict(c.table, mass, c.seq, *a)  # noqa: E731
    for a in ((16, 4, 0, 0), (16, 4, 4, 1), (16, 4, -1, 1), (24, 4, 1, 1), (16, 0, 0, 1)):
        with pytest.raises(RuntimeError):
            evi(*a)
    with pytest.raises(RuntimeError):
        ops.kv8_evict(c.table.long(), mass, c.seq, 16, 4, 1, 1)
