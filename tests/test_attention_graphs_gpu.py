"""Captured attention over the 4-bit cache: graphs captured on one stream and replayed at the same time on two, several
calls in one graph, captures on a stream that ran nothing before."""
import numpy as np
import pytest
import torch

import test_serving_gpu as serving
from test_attention_gpu import _paged, _randn

pytestmark = pytest.mark.gpu
_i32 = serving._i32


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _captured(call, stream):
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    return graph, out


def _replayed(graphs, outs, wants, eager, turns=4):
    """at the same time on streams of their own, with eager calls beside them, and one after the other"""
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(turns):
        for out in outs:
            for x in out:
                x.fill_(-1)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s if turn % 2 == 0 else streams[0]):
                graph.replay()
        beside = eager()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
        assert all(torch.equal(a, b) for a, b in zip(beside, wants[0])), turn


def test_captures_are_told_apart():
    from grinqh import _lib
    lib, side = _lib.load_library(), torch.cuda.Stream()
    ids = []
    for _ in range(3):
        assert lib.grinqh_capture_id(side.cuda_stream) == 0
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.zeros(1, device="cuda")
            ids.append(lib.grinqh_capture_id(side.cuda_stream))
            assert lib.grinqh_capture_id(side.cuda_stream) == ids[-1]
    assert 0 not in ids and len(set(ids)) == 3


@pytest.mark.parametrize("lens,hkv,d", [([9000], 2, 128), ([30000, 500], 1, 64), ([5000, 40, 5000], 2, 256)])
@pytest.mark.parametrize("per_head", [False, True])
def test_two_graphs_of_one_stream_at_once(lens, hkv, d, per_head):
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    cache, table, lengths, _ = _paged(rng, lens, hkv, d, 16, d // 2, "f16")
    table = table.unsqueeze(1).repeat(1, hkv, 1) if per_head else table
    qs = [_randn(rng, len(lens), 4 * hkv, d) for _ in range(2)]
    calls = [lambda q=q: (ga.kv4_attention(q, cache, table, lengths),) for q in qs]
    wants = [call() for call in calls]
    side = torch.cuda.Stream()
    graphs, outs = zip(*[_captured(call, side) for call in calls])
    _replayed(graphs, outs, wants, calls[0])


def test_graphs_of_several_calls():
    """both attentions, several times in a graph, of different sizes: the calls follow each other in one workspace"""
    from grinqh import attention as ga
    rng = np.random.default_rng(4)
    cache, table, lengths, _ = _paged(rng, [9000, 40, 3000], 2, 128, 16, 64, "f16")
    wide = torch.nn.functional.pad(table, (0, 8000), value=-1)
    ends, few = _i32([0, 2, 3, 80]), _i32([0, 300, 300, 310])

    def program(q, rows, more):
        a = ga.kv4_attention(q, cache, table, lengths)
        b = ga.kv4_chunk_attention(rows, cache, table, lengths, ends)
        c = ga.kv4_attention(q * 0.5 + a, cache, table, lengths)
        e = ga.kv4_chunk_attention(more, cache, wide, lengths, few)
        return a, b, c, e, ga.kv4_attention(c, cache, wide, lengths)

    inputs = [(_randn(rng, 3, 8, 128), _randn(rng, 80, 8, 128), _randn(rng, 310, 8, 128)) for _ in range(2)]
    calls = [lambda x=x: program(*x) for x in inputs]
    wants = [call() for call in calls]
    side = torch.cuda.Stream()
    graphs, outs = zip(*[_captured(call, side) for call in calls])
    _replayed(graphs, outs, wants, calls[0])
    del graphs, outs  # a later capture on the same stream, when those graphs' memory is gone
    graph, out = _captured(calls[1], side)
    _replayed([graph], [out], [wants[1]], calls[1])


def test_steps_over_selected_pages_on_two_streams():
    """whole steps whose selected pages are shared by several blocks"""
    rng = np.random.default_rng(5)
    start, count, width = [4000, 30, 2500], 140, 300

    def server(seed):
        g = np.random.default_rng(seed)
        s = serving._Server(g, 3, pages=500, width=width)
        n = sum(start)
        s.step(_randn(g, n, 8, 128), _randn(g, n, 2, 128), _randn(g, n, 2, 128), _i32(start))
        return s

    q, k, v = _randn(rng, 3, 8, 128), _randn(rng, 3, 2, 128), _randn(rng, 3, 2, 128)
    one = _i32([1, 1, 1])
    eager, captured = [server(i) for i in (1, 2)], [server(i) for i in (1, 2)]
    side = torch.cuda.Stream()
    graphs, outs = zip(*[_captured(lambda s=s: s.step(q, k, v, one, count), side) for s in captured])
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(5):
        wants = [s.step(q, k, v, one, count) for s in eager]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, b, out, want in zip(captured, eager, outs, wants):
            assert torch.equal(a.lengths, b.lengths) and torch.equal(a.table, b.table)
            assert torch.equal(out, want), turn


def test_two_streams_of_one_capture():
    """a graph whose calls run beside each other"""
    from grinqh import attention as ga
    rng = np.random.default_rng(6)
    cache, table, lengths, _ = _paged(rng, [9000, 3000], 2, 128, 16, 64, "f16")
    qs = [_randn(rng, 2, 8, 128) for _ in range(2)]
    rows, ends = _randn(rng, 40, 8, 128), _i32([0, 3, 40])

    def program(other):
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            outs = [ga.kv4_attention(qs[0], cache, table, lengths), ga.kv4_chunk_attention(rows, cache, table, lengths, ends)]
        outs += [ga.kv4_attention(qs[1], cache, table, lengths), ga.kv4_chunk_attention(rows, cache, table, lengths, ends)]
        here.wait_stream(other)
        return outs

    want = program(torch.cuda.Stream())
    graph, out = _captured(lambda: program(torch.cuda.Stream()), torch.cuda.Stream())
    _replayed([graph], [out], [want], lambda: program(torch.cuda.Stream()))
