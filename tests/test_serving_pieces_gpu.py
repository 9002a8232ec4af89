"""kv4_chunk_attention where all work is cut into equal pieces, and at the edges of a batch.

Which way a batch is shared out goes by its rows and the table's width (some 48 tiles of 64 tokens for each of 256
blocks), then by the lengths; the results are held against the same definition in 64 bits."""
import numpy as np
import pytest
import torch

import test_serving_gpu as serving

pytestmark = pytest.mark.gpu
_chunk_case, _check_chunk, _i32 = serving._chunk_case, serving._check_chunk, serving._i32


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _wide(table, pages=8000):
    return torch.nn.functional.pad(table, (0, pages), value=-1)


@pytest.mark.parametrize("lens,news", [([9000], [300]), ([9000, 30, 4513], [300, 30, 2]), ([4000, 0, 5000], [129, 0, 400]),
                                       ([0, 8191, 1, 6000], [70, 257, 1, 300]), ([5000, 4992], [260, 600])])
@pytest.mark.parametrize("hkv,per,d", [(2, 4, 128), (3, 17, 64), (3, 2, 256)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_units_are_cut(lens, news, hkv, per, d, dtype):
    """a unit in several pieces: parts of a tile's worth, and no order of blocks changes a result"""
    from grinqh import attention as ga
    case = _chunk_case(d + len(lens), lens, news, hkv, per, d, 16, d // 2, dtype, behind=3, in_front=2)
    cache, table, lengths, kv, q, ends = case
    outs = [ga.kv4_chunk_attention(q, cache, _wide(table), lengths, ends) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    _check_chunk(outs[0], q, kv, news, d // 2, dtype, first=2)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_pieces_with_several_units(d):
    """whole units, ends and beginnings in one piece, more than 64 sequences, some of them with few rows"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    news = rng.integers(66, 90, 80)
    news[[3, 40, 79]] = [1, 0, 5]
    lens = news + rng.integers(0, 40, 80)
    lens[30], news[30], lens[70] = 9000, 300, 5000
    case = _chunk_case(d, lens.tolist(), news.tolist(), 1, 4, d, 16, 64, "f16", behind=4)
    cache, table, lengths, kv, q, ends = case
    outs = [ga.kv4_chunk_attention(q, cache, _wide(table), lengths, ends) for _ in range(2)]
    assert torch.equal(*outs)
    _check_chunk(outs[0], q, kv, news.tolist(), 64, "f16")


@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_in_a_cut_unit(which):
    """a token that is NaN reaches the rows that see it through every part, and no other"""
    from grinqh import attention as ga
    lens, news = [9000, 70], [300, 70]
    cache, table, lengths, kv, q, ends = _chunk_case(8, lens, news, 2, 4, 128, 16, 64, "f16")
    clean = ga.kv4_chunk_attention(q, cache, _wide(table), lengths, ends)
    k, v = (x.clone() for x in kv[0])
    (k if which == "k" else v)[8900] = float("nan")   # rows see it from row 200 on
    slots = table[0].long().repeat_interleave(16)[:9000] * 16 + torch.arange(9000, device="cuda") % 16
    ga.kv4_store(cache, k, v, slots)
    out = ga.kv4_chunk_attention(q, cache, _wide(table), lengths, ends)
    assert torch.equal(out[:200], clean[:200]) and torch.equal(out[300:], clean[300:])
    assert bool(out[200:300].isnan().all())


def test_pieces_with_bad_pages_and_lengths():
    from grinqh import attention as ga
    lens, news = [9000, 5000, 100], [300, 200, 80]
    cache, table, lengths, kv, q, ends = _chunk_case(9, lens, news, 2, 4, 64, 16, 64, "f16")
    wide = _wide(table)
    clean = ga.kv4_chunk_attention(q, cache, wide, lengths, ends)
    for page in (-1, cache.shape[0], -(1 << 31)):
        bad = wide.clone()
        bad[0, 200] = page
        out = ga.kv4_chunk_attention(q, cache, bad, lengths, ends)
        assert bool(out[:300].isnan().all()) and torch.equal(out[300:], clean[300:])
    long = lengths.clone()
    long[1] = wide.shape[1] * 16 + 1
    out = ga.kv4_chunk_attention(q, cache, wide, long, ends)
    assert bool(out[300:500].isnan().all())
    _check_chunk(out[:300], q[:300], kv[:1], news[:1], 64, "f16")
    _check_chunk(out[500:], q[500:], kv[2:], news[2:], 64, "f16")


@pytest.mark.parametrize("rows", [7, 112, 400])
def test_offsets_that_are_not_ascending_leave_the_next_call_right(rows):
    from grinqh import attention as ga
    lens, news = [9000, 3000, 3000], [rows - 6, 4, 2]
    cache, table, lengths, kv, q, ends = _chunk_case(rows, lens, news, 2, 4, 64, 16, 64, "f16")
    for tab in (table, _wide(table)):
        for e in ([0, rows, 3, rows], [rows, 0, rows, 0], [-5, 2 * rows, 1 << 30, -(1 << 31)], [5, 5, 2, 1]):
            ga.kv4_chunk_attention(q, cache, tab, lengths, _i32(e))
            _check_chunk(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, kv, news, 64, "f16")


def test_no_sequences_no_rows_and_no_tokens():
    """rows that belong to no sequence are zeros, also where there is no sequence at all"""
    from grinqh import attention as ga
    cache, table, lengths, kv, q, ends = _chunk_case(1, [40, 40], [3, 30], 2, 4, 128, 16, 64, "f16")
    for x in (q, q[:2], q.repeat(20, 1, 1)):
        for e in ([0], [5], [-1]):
            out = ga.kv4_chunk_attention(x, cache, table[:0], lengths[:0], _i32(e))
            assert out.shape == x.shape and not out.any()
        for tab in (table, _wide(table)):
            assert not ga.kv4_chunk_attention(x, cache, tab, lengths * 0, ends).any()
    assert ga.kv4_chunk_attention(q[:0], cache, table, lengths, ends * 0).shape == (0, 8, 128)


@pytest.mark.parametrize("rows", [40, 300])
def test_two_graphs_at_once_and_eager_calls_between(rows):
    """captured calls have counters and parts of their own: replays on two streams do not meet"""
    from grinqh import attention as ga
    lens, news = [9000, 700], [rows, 100]
    cache, table, lengths, kv, q, ends = _chunk_case(rows, lens, news, 2, 4, 128, 16, 64, "f16")
    wide = _wide(table)
    want = ga.kv4_chunk_attention(q, cache, wide, lengths, ends)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(ga.kv4_chunk_attention(q, cache, wide, lengths, ends))
        graphs.append(graph)
    for _ in range(4):
        for out in outs:
            out.fill_(-1)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = ga.kv4_chunk_attention(q, cache, wide, lengths, ends)
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in (*outs, eager))


def test_tables_without_pages():
    """no room for any token: rows see none, and a length is past the table"""
    from grinqh import attention as ga
    cache, table, lengths, kv, q, ends = _chunk_case(5, [40, 40], [3, 200], 2, 4, 128, 16, 64, "f16")
    for x, e in ((q, ends), (q[:5], _i32([0, 3, 5]))):
        assert not ga.kv4_chunk_attention(x, cache, table[:, :0], lengths * 0, e).any()
        assert bool(ga.kv4_chunk_attention(x, cache, table[:, :0], lengths, e).isnan().all())


@pytest.mark.parametrize("per,d", [(65, 64), (128, 128), (130, 256)])
def test_more_heads_per_key_head_than_rows_of_a_block(per, d):
    """one token is more rows than the single-token kernel or the tile kernel takes in a block"""
    from grinqh import attention as ga
    lens, news = [300, 5, 1, 70], [1, 5, 1, 9]
    cache, table, lengths, kv, q, ends = _chunk_case(per, lens, news, 1, per, d, 16, d, "bf16")
    for tab in (table, _wide(table)):
        _check_chunk(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, kv, news, d, "bf16")


@pytest.mark.parametrize("new", [2, 90])
def test_sequences_that_share_pages(new):
    """one prefix, several questions: the same pages in several rows of the table"""
    from grinqh import attention as ga
    case = _chunk_case(new, [400], [new], 2, 4, 128, 16, 64, "f16")
    cache, table, lengths, kv, q, ends = case
    want = ga.kv4_chunk_attention(q, cache, _wide(table), lengths, ends)
    _check_chunk(want, q, kv, [new], 64, "f16")
    n = 5
    out = ga.kv4_chunk_attention(q.repeat(n, 1, 1), cache, _wide(table).expand(n, -1), lengths.expand(n),
                                 _i32(np.arange(n + 1) * new))
    _check_chunk(out, q.repeat(n, 1, 1), kv * n, [new] * n, 64, "f16")
