"""The operators of the 8-bit cache in CUDA graphs and on several streams: a graph's replay depends on no call outside it,
whatever was captured or called before, after or at the same time.  Every result is compared bit for bit with that of a
plain call, since the sums run in a fixed order."""
import pytest
import torch

from mfd_b200 import ops
from mfd_b200._lib import CaptureScratch, Workspace
from test_gpu_kv8 import DEV, Case

pytestmark = pytest.mark.gpu


def _attend(c):
    kw = dict(k_new=c.kn, v_new=c.vn, anc=c.anc(), return_lse=True)
    return lambda: ops.kv8_attention(c.q, c.k, c.v, c.ks, c.vs, c.table, c.seq, c.scale, **kw)


def _weigh(c):
    lse = _attend(c)()[1]
    mass = torch.rand(c.table.shape, device=DEV)
    return lambda: (ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, mass, decay=0.5),)


def _capture(call, **kw):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, **kw):
        got = call()
    return graph, got


def _same(got, want):
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _wipe(got):
    for t in got:
        t.fill_(7.0)


# one request in many pieces (tickets and partials), a batch, and trees (the combination's partials)
SHAPES = [dict(lens=[9000], n=1, heads=8, kv=2, page=64), dict(lens=[700, 64, 0, 333, 2100], n=2, heads=8, kv=2, page=32),
          dict(lens=[3000, 40], n=40, heads=8, kv=2, page=32)]


@pytest.mark.parametrize("make", [_attend, _weigh])
@pytest.mark.parametrize("first,second", [(0, 1), (1, 0), (2, 0), (0, 2), (1, 1)])
def test_two_graphs_of_the_default_capture_stream_in_any_order(make, first, second):
    """torch.cuda.graph's own stream, on which nothing was called before; the graph captured second is replayed first."""
    calls = [make(Case(200 + i, **SHAPES[i], stale=False)) for i in (first, second)]
    want = [tuple(t.clone() for t in call()) for call in calls]
    graphs = [_capture(call) for call in calls]
    for i in (1, 0, 1, 1, 0):
        _wipe(graphs[i][1])
        graphs[i][0].replay()
        _same(graphs[i][1], want[i])


@pytest.mark.parametrize("make", [_attend, _weigh])
def test_graphs_of_one_capture_stream_replayed_on_two_streams_at_once(make):
    calls = [make(Case(210 + i, **SHAPES[i], stale=False)) for i in (0, 2)]
    want = [tuple(t.clone() for t in call()) for call in calls]
    graphs = [_capture(call) for call in calls]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(100):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    for (_, got), w in zip(graphs, want):
        _same(got, w)


@pytest.fixture(autouse=True, params=["spare tickets", "none"])
def _spare(request, monkeypatch):
    """With the tickets that plain calls leave for captures, and where they are used up (the graph zeroes its own)."""
    if request.param == "none":
        monkeypatch.setattr(CaptureScratch, "_spare", {0: (torch.zeros(0, dtype=torch.uint8, device=DEV), 0)})


def _forget():
    torch.cuda.synchronize()
    for key in [k for k in Workspace._cache if isinstance(k[1], tuple) and str(k[1][0]).startswith("kv8")]:
        del Workspace._cache[key]
    CaptureScratch._held.clear()


@pytest.mark.parametrize("warm", [True, False])
def test_a_graph_stays_right_beside_larger_and_smaller_calls_on_its_stream(warm):
    """A decode step is captured; calls with more rows and more requests on the same stream then grow the scratch of plain
    calls, and memory that was given back is written by others."""
    _forget()
    small, large = Case(220, **SHAPES[0], stale=False), Case(221, [300] * 300, n=9, heads=8, kv=2, page=32, stale=False)
    step, tree = _attend(small), _attend(large)
    want, want_tree = step(), tree()
    _forget()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(side):
            step()
    torch.cuda.synchronize()
    graph, got = _capture(step, stream=side)
    for _ in range(3):
        with torch.cuda.stream(side):
            again = tree()
            others = [torch.full((1 << k,), 0x5A, dtype=torch.uint8, device=DEV) for k in range(8, 25) for _ in range(4)]
        _wipe(got)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
            small_again = step()
        _same(got, want)
        _same(small_again, want)
        _same(again, want_tree)
        assert all(bool((t == 0x5A).all()) for t in others)
        del others


def test_calls_of_different_sizes_in_one_graph_and_on_two_of_its_streams():
    cases = [Case(230 + i, **s, stale=False) for i, s in enumerate(SHAPES)]
    calls = [_attend(c) for c in cases] + [_weigh(cases[1])]
    want = [tuple(t.clone() for t in call()) for call in calls]

    def all_of_them():
        main, side = torch.cuda.current_stream(), torch.cuda.Stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            there = [calls[i]() for i in (2, 0)]
        here = [calls[i]() for i in (0, 1, 2, 3, 1)]
        main.wait_stream(side)
        return there + here

    graph, got = _capture(all_of_them)
    for _ in range(3):
        for out in got:
            _wipe(out)
        graph.replay()
        for out, i in zip(got, (2, 0, 0, 1, 2, 3, 1)):
            _same(out, want[i])


def test_graphs_in_a_shared_pool_replayed_in_order():
    calls = [_attend(Case(240 + i, **SHAPES[i], stale=False)) for i in (2, 0, 1)]
    want = [tuple(t.clone() for t in call()) for call in calls]
    graphs = [_capture(calls[0])]
    for call in calls[1:]:
        graphs.append(_capture(call, pool=graphs[0][0].pool()))
    for _ in range(2):
        for (graph, got), w in zip(graphs, want):
            graph.replay()
            _same(got, w)


@pytest.mark.parametrize("make", [_attend, _weigh])
def test_streams_at_once(make):
    call = make(Case(250, **SHAPES[1], stale=False))
    want = call()
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [call() for _ in range(20)]
    for out in outs:
        _same(out, want)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_a_captured_append_goes_on_from_where_the_cache_is(dtype):
    """Ten replays of append, page weights and attention, the lengths fed back, against ten plain steps."""
    def steps(replay):
        c = Case(260, [5, 60, 0], n=6, heads=8, kv=2, page=16, dtype=dtype, spare=60, stale=False)
        mass = torch.zeros(c.table.shape, device=DEV)
        attend = _attend(c)

        def step():
            out, lse = attend()
            ops.kv8_page_weights(c.q, lse, c.k, c.ks, c.table, c.seq, c.scale, mass, decay=0.9, out=mass)
            c.seq.copy_(ops.kv8_append(c.k, c.v, c.ks, c.vs, c.kn, c.vn, c.table, c.seq))
            return out, lse

        if not replay:
            for _ in range(10):
                got = step()
        else:
            graph, got = _capture(step)
            for _ in range(10):
                graph.replay()
        torch.cuda.synchronize()
        return (*got, c.seq, mass, c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)

    want = steps(False)
    assert want[2].tolist() == [65, 120, 60]
    _same(steps(True), want)
    assert ops.kv8_attention_status() == 0
