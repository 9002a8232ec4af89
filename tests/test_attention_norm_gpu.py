"""Attention over the 4-bit cache against its definition in 64 bits, by the norm of the error: how
work that is split, cut or shared out between kernels is put together again (_attention_norm.py)."""
import numpy as np
import pytest
import torch

import _attention_norm as norm
import test_serving_gpu as serving
from test_attention_gpu import _paged, _randn

pytestmark = pytest.mark.gpu
_chunk_case, _i32 = serving._chunk_case, serving._i32


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _wide(table, pages=8000):
    """with room for far more tokens: the single-token kernel then has 64 rows of a sequence at most, and long units are
    cut into pieces"""
    return torch.nn.functional.pad(table, (0, pages), value=-1)


def _chunk(lens, news, hkv, per, d, group, dtype, seed=0, tables=None, page=16):
    from grinqh import attention as ga
    case = _chunk_case(seed + d + sum(news), lens, news, hkv, per, d, page, group, dtype, behind=3, in_front=2)
    cache, table, lengths, kv, q, ends = case
    for tab in (table, _wide(table)) if tables is None else tables(table):
        norm.check(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, kv, news, group, dtype, first=2)


@pytest.mark.parametrize("lens,news", [([2777], [3]), ([2777], [40]), ([9000, 1, 513], [2, 1, 1]),
                                       ([9000, 30, 4513], [70, 30, 2]), ([4000, 0, 5000], [129, 0, 400])])
@pytest.mark.parametrize("hkv,per,d,dtype", [(2, 4, 128, "f16"), (1, 17, 64, "bf16"), (3, 1, 256, "f16")])
def test_split_units(lens, news, hkv, per, d, dtype):
    _chunk(lens, news, hkv, per, d, d // 2, dtype)


@pytest.mark.parametrize("lens,news", [([9000], [300]), ([9000, 30, 4513], [300, 30, 2]), ([4000, 0, 5000], [129, 0, 400]),
                                       ([0, 8191, 1, 6000], [70, 257, 1, 300]), ([5000, 4992], [260, 600])])
@pytest.mark.parametrize("hkv,per,d,dtype", [(2, 4, 128, "f16"), (2, 4, 128, "bf16"), (3, 17, 64, "f16"),
                                             (3, 2, 256, "bf16")])
def test_cut_units(lens, news, hkv, per, d, dtype):
    _chunk(lens, news, hkv, per, d, d // 2, dtype, tables=lambda t: [_wide(t)])


@pytest.mark.parametrize("length", [4095, 4096, 4097, 4159, 4161, 6016])
@pytest.mark.parametrize("new", [5, 64, 127, 256])
def test_lengths_around_tiles(length, new):
    _chunk([length, length // 2], [new, new], 2, 4, 64, 64, "f16")


@pytest.mark.parametrize("seqs,lead", [(63, 90), (80, 300), (700, 1)])
def test_many_sequences(seqs, lead):
    rng = np.random.default_rng(seqs)
    news = rng.integers(0, 3, seqs) if seqs != 80 else rng.integers(60, 90, seqs)
    lens = news + rng.integers(0, 60, seqs)
    news[seqs // 3], lens[seqs // 3] = lead, 9000
    news[-1], lens[-1] = lead, 700
    _chunk(lens.tolist(), news.tolist(), 1, 4, 128, 64, "f16")


@pytest.mark.parametrize("d,group", [(64, 32), (128, 128), (256, 64)])
def test_rows_that_look_for_one_token(d, group):
    """row i's query is a token's own key, at the ends of tiles and up to the row's own token: its value is the result"""
    from grinqh import attention as ga
    length, rows = 9000, 300
    cache, table, lengths, kv, q, ends = _chunk_case(d, [length], [rows], 1, 4, d, 16, group, "f16")
    k = kv[0][0]
    for shift in (-1, 0, 1):
        target = (64 * (torch.arange(rows * 4) * 7 % 136) + shift).clamp(0, length - rows)
        target[::9] = (torch.arange(rows * 4) // 4 + length - rows)[::9]
        q.copy_((k[target.cuda(), 0] * (40.0 * d ** 0.5 / k.float().pow(2).sum(-1).mean())).view(rows, 4, d))
        kept = norm.kept(k, group), norm.kept(kv[0][1], d)
        want = norm.definition(q, *kept)
        most = norm.worst(q, *kept, "f16", want)
        assert float((most / want.pow(2).sum(-1).sqrt()).mean()) < 0.1  # another token's value is past that
        for tab in (table, _wide(table)):
            out = ga.kv4_chunk_attention(q, cache, tab, lengths, ends).double().cpu()
            assert bool(((out - want).pow(2).sum(-1).sqrt() <= most).all())


@pytest.mark.parametrize("lens", [[9000], [20000, 40, 0, 513], [1, 31, 33, 5000, 4097]])
@pytest.mark.parametrize("hkv,per,d,dtype", [(2, 4, 128, "f16"), (1, 17, 64, "bf16"), (3, 1, 256, "f16")])
def test_single_tokens(lens, hkv, per, d, dtype):
    """kv4_attention, over one table for all heads and over one per head"""
    from grinqh import attention as ga
    rng = np.random.default_rng(len(lens) + d)
    cache, table, lengths, kv = _paged(rng, lens, hkv, d, 16, d // 2, dtype)
    q = _randn(rng, len(lens), hkv * per, d, dtype=dtype)
    for tab in (table, _wide(table, 700), table.unsqueeze(1).repeat(1, hkv, 1)):
        norm.check(ga.kv4_attention(q, cache, tab, lengths), q, kv, [1] * len(lens), d // 2, dtype)


@pytest.mark.parametrize("count", [40, 300])
def test_single_tokens_over_selected_pages(count):
    from grinqh import attention as ga
    rng = np.random.default_rng(count)
    page, hkv, per = 16, 2, 4
    lens = [9000, 5001, 100]
    cache, table, lengths, kv = _paged(rng, lens, hkv, 128, page, 64, "f16")
    summary = ga.kv4_summary(cache)
    ga.kv4_summarize(cache, summary, table, torch.zeros_like(lengths), lengths)
    q = _randn(rng, 3, hkv * per, 128)
    pages, some = ga.kv4_select(q, summary, table, lengths, page, count)
    out = ga.kv4_attention(q, cache, pages, some)
    for i, n in enumerate(lens):
        place = {int(x): j for j, x in enumerate(table[i, :-(-n // page)].tolist())}
        for h in range(hkv):
            at = torch.cat([torch.arange(place[x] * page, min(place[x] * page + page, n))
                            for x in pages[i, h].tolist() if x >= 0]).cuda()
            assert len(at) == int(some[i])
            heads = slice(h * per, (h + 1) * per)
            norm.check(out[i:i + 1, heads], q[i:i + 1, heads], [tuple(x[at, h:h + 1] for x in kv[i])], [1], 64, "f16")
