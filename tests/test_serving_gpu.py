"""GPU tests of the operators around the 4-bit cache (csrc/append.hip,
csrc/chunk.hip, csrc/select.hip, grinqh/attention.py): room for new tokens,
attention of chunks, page summaries, the selection by them and the attention
over selected pages.

Everything but the attentions is exact: integers, and floats that are sums
without rounding.  A chunk's results are held to the worst case of its
arithmetic: keys, values and weights are fp16 (2^-11 of their size each; the
weights' error counts twice, in the sum and in its divisor), a logit is off by
2^-11 of the magnitudes it sums for its keys' rounding and 2^-20 for fp32, and
that counts twice in the exponential and its divisor; then one rounding of the
result.  Weights below fp16's normal range are off by 2^-25 beside a largest
weight of 1 at least."""
import math

import numpy as np
import pytest
import torch

from test_attention_gpu import DT, LAYOUTS, LIMIT, U, _check_decode, _paged, _params, _quantize, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


# ---------------------------------------------------------------- chunks

def _check_chunk(out, q, seqs, news, group, dtype, scale=None, first=0):
    """out [rows, heads, d] against fp64: sequence i has news[i] rows, its keys and values are seqs[i] [T, H, D]"""
    out, qf = out.double().cpu().numpy(), q.double().cpu().numpy()
    d = qf.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    at = first
    assert not out[:first].any()
    for i, ((k, v), rows) in enumerate(zip(seqs, news)):
        t, hkv, _ = k.shape
        per = qf.shape[1] // hkv
        if rows and t:
            ks, km = _params(k.float().cpu().numpy(), group)
            vs, vm = _params(v.float().cpu().numpy(), d)
            seen = np.arange(t)[None] <= np.arange(rows)[:, None] + t - rows
        for h in range(hkv if rows else 0):
            got = out[at:at + rows, h * per:(h + 1) * per]
            if t == 0:
                assert not got.any()
                continue
            qh = qf[at:at + rows, h * per:(h + 1) * per]
            s = np.where(seen[:, None], qh @ (ks + km)[:, h].T * scale, -np.inf)
            some = seen.any(-1)
            assert not got[~some].any()
            s, qh, got = s[some], qh[some], got[some]
            if not len(s):
                continue
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o = p @ (vs + vm)[:, h]
            size = (np.abs(qh) @ (np.abs(km) + ks)[:, h].T * scale).max(-1, keepdims=True)
            delta = (2.0 ** -11 + 2.0 ** -20) * size + 2.0 ** -20
            big = (np.abs(vm) + vs)[:, h]
            tol = ((3 * U["f16"] + 2 * delta + 2.0 ** -17) * (p @ big) + U[dtype] * np.abs(o)
                   + t * 2.0 ** -25 * big.max() + 2.0 ** -24)
            err = np.abs(got - o)
            assert (err <= tol).all(), (i, h, float((err / tol).max()))
        at += rows
    assert not out[at:].any()


def _chunk_case(seed, lens, news, hkv, per, d, page, group, dtype, behind=0, in_front=0):
    rng = np.random.default_rng(seed)
    cache, table, lengths, seqs = _paged(rng, lens, hkv, d, page, group, dtype)
    q = _randn(rng, in_front + sum(news) + behind, hkv * per, d, dtype=dtype)
    ends = _i32(np.cumsum([in_front] + list(news)))
    return cache, table, lengths, seqs, q, ends


def _tables(table):
    """The table, and one with room for far more: which kernel serves a sequence goes by its rows and by the table's
    width (64 rows at most go to the single-token kernel where the table is wide, 256 where it is narrow)."""
    return table, torch.nn.functional.pad(table, (0, 8000), value=-1)


@pytest.mark.parametrize("dtype,d,group,page,hkv", LAYOUTS)
@pytest.mark.parametrize("per", [1, 4, 7])
@pytest.mark.parametrize("kind", ["few", "both", "one"])
def test_chunk(dtype, d, group, page, hkv, per, kind):
    """few rows per sequence, many and few together, a single sequence: the three ways a batch is served"""
    from grinqh import attention as ga
    if kind == "few":
        lens, news = [0, 1, 2, 16, 31, 33, 64, 200, 500, 7], [0, 1, 2, 1, 2, 1, 0, 2, 1, 3]
    elif kind == "both":
        lens, news = [170, 164, 65, 227, 300, 40, 5, 0, 700, 33], [170, 1, 64, 130, 299, 1, 5, 3, 64 // per, 0]
    else:
        lens, news = [413], [150]
    case = _chunk_case(d + group + per, lens, news, hkv, per, d, page, group, dtype, behind=5, in_front=3)
    cache, table, lengths, seqs, q, ends = case
    for tab in _tables(table):
        out = ga.kv4_chunk_attention(q, cache, tab, lengths, ends)
        _check_chunk(out, q, seqs, news, group, dtype, first=3)


@pytest.mark.parametrize("per", [16, 17, 40])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_many_query_heads(per, d):
    from grinqh import attention as ga
    for lens, news in (([70, 3, 333], [1, 3, 20]), ([200], [21])):
        cache, table, lengths, seqs, q, ends = _chunk_case(per, lens, news, 2, per, d, 32, 64, "f16")
        for tab in _tables(table):
            _check_chunk(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, seqs, news, 64, "f16")


@pytest.mark.parametrize("lens,news", [([2777], [3]), ([2777], [40]), ([9000, 1, 513], [2, 1, 1]),
                                       ([9000, 30, 4513], [70, 30, 2]), ([4000, 0, 5000], [129, 0, 400])])
@pytest.mark.parametrize("hkv,per,d", [(2, 4, 128), (1, 17, 64), (3, 1, 256)])
def test_chunk_split_lengths(lens, news, hkv, per, d):
    """few units are shared by several blocks; a table with room for more changes nothing but the plan"""
    from grinqh import attention as ga
    cache, table, lengths, seqs, q, ends = _chunk_case(17, lens, news, hkv, per, d, 16, d // 2, "bf16")
    wide = torch.nn.functional.pad(table, (0, 700), value=-1)
    for tab in (table, wide):
        outs = [ga.kv4_chunk_attention(q, cache, tab, lengths, ends) for _ in range(2)]
        assert torch.equal(*outs)  # the counters are zero again after a call, and no order changes a result
        _check_chunk(outs[0], q, seqs, news, d // 2, "bf16")


@pytest.mark.parametrize("seqs", [62, 63, 64, 130, 700])
@pytest.mark.parametrize("lead", [1, 90])
def test_chunk_many_sequences(seqs, lead):
    from grinqh import attention as ga
    rng = np.random.default_rng(seqs)
    news = rng.integers(0, 3, seqs)
    lens = news + rng.integers(0, 60, seqs)
    news[seqs // 3], lens[seqs // 3] = lead, 3000
    news[-1], lens[-1] = lead, 700
    case = _chunk_case(seqs, lens.tolist(), news.tolist(), 1, 2, 64, 16, 64, "f16", behind=100, in_front=1)
    cache, table, lengths, kv, q, ends = case
    for tab in (table, torch.nn.functional.pad(table, (0, 1000), value=-1)):
        _check_chunk(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, kv, news.tolist(), 64, "f16", first=1)


def test_chunk_fewer_tokens_than_rows():
    """rows are aligned with the last tokens: the first ones may see none"""
    from grinqh import attention as ga
    lens, news = [40, 3, 0, 64, 5], [100, 8, 70, 64, 30]
    cache, table, lengths, seqs, q, ends = _chunk_case(4, lens, news, 2, 4, 128, 16, 32, "f16")
    for tab in _tables(table):
        _check_chunk(ga.kv4_chunk_attention(q, cache, tab, lengths, ends), q, seqs, news, 32, "f16")


@pytest.mark.parametrize("news", [[4, 2], [150, 2]])
@pytest.mark.parametrize("which", ["k", "v"])
def test_chunk_nan_reaches_only_rows_that_see_it(news, which):
    from grinqh import attention as ga
    lens = [300, 50]
    cache, table, lengths, kv, q, ends = _chunk_case(6, lens, news, 2, 4, 128, 16, 64, "f16")
    table = _tables(table)[1]
    clean = ga.kv4_chunk_attention(q, cache, table, lengths, ends)
    row = news[0] - 2                       # the last row but one
    token = lens[0] - news[0] + row         # its own token
    k, v = (x.clone() for x in kv[0])
    (k if which == "k" else v)[token, 1, 3] = float("nan")
    slot = table[0, token // 16].long() * 16 + token % 16
    ga.kv4_store(cache, k[token:token + 1], v[token:token + 1], slot.view(1))
    out = ga.kv4_chunk_attention(q, cache, table, lengths, ends)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[row:news[0], 4:] = True             # second key/value head's query heads
    assert bool(out[hit].isnan().all())
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [2, 70])
def test_chunk_values_at_the_limit(dtype, new):
    """codes that stand for more than fp16 holds, fp16 results that stay finite, keys of the same size"""
    from grinqh import attention as ga
    rng = np.random.default_rng(9)
    n = 200
    k = _randn(rng, n, 1, 128, dtype=dtype)
    v = torch.full((n, 1, 128), LIMIT if dtype == "f16" else 1e6, dtype=DT[dtype], device="cuda")
    v[:, :, ::2] = _randn(rng, n, 1, 64, dtype=dtype) * 1000
    k[:, :, 5] = 7e4 if dtype == "bf16" else LIMIT
    cache = ga.kv4_cache(13, 1, 128, 16, 32)
    table = _tables(_i32([[12 - i for i in range(13)]]))[1]
    at = torch.arange(n).cuda()
    ga.kv4_store(cache, k, v, table[0, at // 16].long() * 16 + at % 16)
    q = _randn(rng, new, 4, 128, dtype=dtype)
    q[:, :, 5] *= 1e-5
    out = ga.kv4_chunk_attention(q, cache, table, _i32([n]), _i32([0, new]))
    assert bool(out.isfinite().all())
    got, want = out.float()[:, :, 1::2], float(LIMIT)
    assert float((got - want).abs().max()) <= 2.0 ** -8 * want
    kf, vf = ga.kv4_load(cache, table[0, at // 16].long() * 16 + at % 16, torch.bfloat16)
    assert bool(kf.isfinite().all()) and bool(vf.isfinite().all())


@pytest.mark.parametrize("new", [3, 50])
@pytest.mark.parametrize("size", [0.0, 1e-7, 30.0, 1e4])
def test_chunk_query_sizes_and_scale(new, size):
    from grinqh import attention as ga
    lens, news = [90, 1000], [new, new]
    cache, table, lengths, kv, q, ends = _chunk_case(5, lens, news, 2, 4, 128, 16, 32, "f16")
    table = _tables(table)[1]
    q = q * size
    scale = 0.5 / max(1.0, size)
    _check_chunk(ga.kv4_chunk_attention(q, cache, table, lengths, ends, scale=scale), q, kv, news, 32, "f16", scale)
    qb = q.bfloat16() * (size * 1e-25)
    _check_chunk(ga.kv4_chunk_attention(qb, cache, table, lengths, ends), qb, kv, news, 32, "bf16")


@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("size", [1e6, 1e20, 1e30])
def test_chunk_logits_of_any_size(new, size):
    """One token's key is the query's own direction and wins by far: its value is the result, whatever the logits' size.
    One whose logit is the same must count as much."""
    from grinqh import attention as ga
    rng = np.random.default_rng(8)
    n = 130
    k = _randn(rng, n, 1, 64, dtype="bf16") * 0.01
    v = _randn(rng, n, 1, 64, dtype="bf16")
    k[7, 0, :], k[71, 0, :] = 1.0, 1.0
    cache = ga.kv4_cache(9, 1, 64, 16, 64)
    slots = torch.arange(n).cuda()
    ga.kv4_store(cache, k, v, slots)
    _, kept = ga.kv4_load(cache, slots, torch.bfloat16)
    q = torch.full((new, 2, 64), size, dtype=torch.bfloat16, device="cuda")
    out = ga.kv4_chunk_attention(q, cache, _tables(_i32([list(range(9))]))[1], _i32([n]), _i32([0, new]))
    # a row that ends in front of the second one (the first of 60: it sees 70 + 1 tokens) has the first one's value
    both = (torch.arange(n - new, n) >= 71).cuda().view(-1, 1, 1)
    want = torch.where(both, (kept[7].float() + kept[71].float()) / 2, kept[7].float())
    err = (out.float() - want).abs()
    # bf16 roundings of the two values and of the result, fp16's of the weights and values
    assert bool((err <= 2.0 ** -8 * (kept[7].float().abs() + kept[71].float().abs()) + 2.0 ** -8 * want.abs()).all())


def test_chunk_bad_pages_and_lengths():
    """a page outside the cache: NaN where it is seen, and no other sequence is touched; a length past the table: NaN"""
    from grinqh import attention as ga
    for news in ([3, 2, 1], [60, 70, 2]):
        lens = [200, 150, 40]
        cache, table, lengths, kv, q, ends = _chunk_case(3, lens, news, 2, 4, 128, 16, 128, "f16")
        if news[0] > 16:
            table = _tables(table)[1]
        clean = ga.kv4_chunk_attention(q, cache, table, lengths, ends)
        for page in (-1, cache.shape[0], 2 ** 31 - 1):
            bad = table.clone()
            bad[1, 0] = page
            out = ga.kv4_chunk_attention(q, cache, bad, lengths, ends)
            rows = slice(news[0], news[0] + news[1])
            assert bool(out[rows].isnan().all())
            assert torch.equal(out[:news[0]], clean[:news[0]]) and torch.equal(out[rows.stop:], clean[rows.stop:])
        long = lengths.clone()
        long[0] = table.shape[1] * 16 + 1
        out = ga.kv4_chunk_attention(q, cache, table.clamp_min(0), long, ends)
        assert bool(out[:news[0]].isnan().all())
        # the other sequences' work is shared out differently beside a long one: the same within the bounds
        _check_chunk(out[news[0]:], q[news[0]:], kv[1:], news[1:], 128, "f16")
        none = ga.kv4_chunk_attention(q, cache[:0], table, lengths, ends)
        assert bool(none.isnan().all())


def test_chunk_offsets_that_are_not_ascending_stay_in_bounds():
    """no result is promised, but nothing else is touched and the next call is right"""
    from grinqh import attention as ga
    lens, news = [3000, 3000, 3000], [40, 2, 70]
    cache, table, lengths, kv, q, ends = _chunk_case(2, lens, news, 2, 4, 64, 16, 64, "f16")
    table = _tables(table)[1]
    for e in ([0, 112, 3, 112], [112, 0, 112, 0], [-5, 200, 1 << 30, -(1 << 31)], [50, 50, 2, 1]):
        ga.kv4_chunk_attention(q, cache, table, lengths, _i32(e))
    for few in (q[:7], q):
        e = [0, 2, 4, 7] if len(few) == 7 else [0, 40, 42, 112]
        out = ga.kv4_chunk_attention(few, cache, table, lengths, _i32(e))
        _check_chunk(out, few, kv, np.diff(e).tolist(), 64, "f16")


def test_chunk_strides_and_streams():
    """slices of a fused projection, rows off the alignment, a strided table, another stream than the tensors'"""
    from grinqh import attention as ga
    lens, news = [300, 50, 90], [40, 1, 7]
    cache, table, lengths, kv, q, ends = _chunk_case(12, lens, news, 2, 4, 128, 16, 32, "f16")
    table = _tables(table)[1]
    want = ga.kv4_chunk_attention(q, cache, table, lengths, ends)
    wide = torch.randn((48, 12 * 128 + 8), device="cuda").half()
    wide[:, 8:8 + 1024] = q.flatten(1)
    strided = torch.stack((table, table), 2)[:, :, 0]
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (wide[:, 8:8 + 1024].unflatten(1, (8, 128)), odd, turned):
        assert torch.equal(ga.kv4_chunk_attention(x, cache, strided, lengths, ends), want)
    padded = torch.nn.functional.pad(table, (0, 5), value=-3)[:, :table.shape[1]]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ga.kv4_chunk_attention(q, cache, padded, lengths, ends))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in outs)


def test_chunk_past_32_bit_offsets():
    from grinqh import attention as ga
    rng = np.random.default_rng(11)
    pages = (5 << 30) // (8 * 2176)
    cache = torch.empty((pages, 8, 1, 2176), dtype=torch.uint8, device="cuda")
    n = 100
    table = _i32([[pages - 1 - i for i in range(7)]])
    at = torch.arange(n).cuda()
    k, v = (_randn(rng, n, 8, 128) for _ in (0, 1))
    ga.kv4_store(cache, k, v, table[0, at // 16].long() * 16 + at % 16)
    for new in (2, 30):
        q = _randn(rng, new, 32, 128)
        out = ga.kv4_chunk_attention(q, cache, table, _i32([n]), _i32([0, new]))
        _check_chunk(out, q, [(k, v)], [new], 128, "f16")
    summary = ga.kv4_summary(cache)
    ga.kv4_summarize(cache, summary, table, _i32([0]), _i32([n]))
    want = _summary_ref([k], [n], 128, 16)[0]
    got = summary[table[0].long()].cpu().numpy()
    assert np.array_equal(got[:, :, :128], want[0]) and np.array_equal(_steps(got, 128), want[1])


# ---------------------------------------------------------------- room for new tokens

def _append_ref(table, lengths, counts, free, page, tokens):
    table = [list(r) for r in table]
    free = list(free)
    width = len(table[0]) if table else 0
    slots, positions, ends, after = [], [], [0], []
    for row, n, c in zip(table, lengths, counts):
        n, c = max(n, 0), min(max(c, 0), tokens - ends[-1])
        # a page that is missing is counted as taken: the list of free pages is empty then anyway
        for place in range(-(-n // page), min(-(-(n + c) // page), width)):
            row[place] = free.pop() if free else -1
        for i in range(n, n + c):
            index = row[i // page] if i // page < width else -1
            slots.append(index * page + i % page if index >= 0 else -1)
            positions.append(i)
        ends.append(ends[-1] + c)
        after.append(n + c)
    pad = tokens - len(slots)
    return slots + [-1] * pad, positions + [0] * pad, ends, after, [len(free)], table


def _check_append(table, lengths, counts, free, free_count, page, tokens, spare=0):
    from grinqh import attention as ga
    t = _i32(table).view(len(lengths), -1)
    wide = torch.nn.functional.pad(t, (0, spare), value=77)
    view = wide[:, :t.shape[1]]
    given = [_i32(x) for x in (lengths, counts, free, [free_count])]
    kept = [x.clone() for x in given]
    got = ga.kv4_append(view, *given, page, tokens)
    want = _append_ref(table, lengths, counts, free[:max(min(free_count, len(free)), 0)], page, tokens)
    for name, a, b in zip(got._fields, got, want):
        assert a.tolist() == b, name
    assert view.tolist() == [list(r) for r in want[5]]
    assert bool((wide[:, t.shape[1]:] == 77).all())
    assert all(torch.equal(a, b) for a, b in zip(given, kept))
    return got


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("seqs", [1, 2, 63, 255, 256, 257, 700])
def test_append(page, seqs):
    rng = np.random.default_rng(seqs + page)
    width = 9
    lengths = rng.integers(0, 4 * page, seqs)
    counts = rng.choice([0, 1, 1, 2, 17, 3 * page], seqs)
    lengths[0], counts[0] = page, 1         # a full page: the token opens the next one
    lengths[-1], counts[-1] = 0, page + 1
    table = rng.permutation(seqs * width + 100)[:seqs * width].reshape(seqs, width)
    free = rng.permutation(5000)[:seqs * 5 + 3].tolist()
    total = int(counts.sum())
    for tokens in (total + 11, total):
        _check_append(table.tolist(), lengths.tolist(), counts.tolist(), free, len(free) - 1, page, tokens, spare=3)


def test_append_at_its_limits():
    """no tokens, no sequences, pages that run out, a table that ends, a buffer that ends, negative numbers"""
    from grinqh import attention as ga
    t = [[5, -1, -1], [6, 7, -1], [8, -1, -1]]
    _check_append(t, [16, 20, 3], [0, 0, 0], [1, 2], 2, 16, 0)
    _check_append(t, [16, 20, 3], [0, 0, 0], [1, 2], 2, 16, 4)
    _check_append(t, [16, 20, 3], [5, 30, 20], [1, 2], 2, 16, 60)       # pages run out in the last sequence
    _check_append(t, [16, 20, 3], [5, 30, 20], [1, 2, 3], 0, 16, 60)    # none at all
    _check_append(t, [16, 20, 3], [5, 30, 20], [1, 2, 3], -9, 16, 60)
    _check_append(t, [16, 20, 3], [5, 30, 20], [1, 2, 3], 99, 16, 60)   # more than the list holds
    _check_append(t, [16, 20, 3], [50, 1, 100], [10, 11, 12, 13, 14, 15, 16], 7, 16, 200)  # past the table
    _check_append(t, [16, 20, 3], [5, 30, 20], [1, 2, 3, 4, 5], 5, 16, 17)  # the buffer ends inside a sequence
    _check_append(t, [-4, 20, 3], [5, -30, 20], [1, 2, 3, 4, 5], 5, 16, 40)
    _check_append([[], [], []], [0, 16, 3], [5, 1, 20], [1, 2, 3, 4, 5], 5, 16, 40)  # a table without room
    none = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    got = ga.kv4_append(none, _i32([]), _i32([]), _i32([3]), _i32([1]), 16, 3)
    assert [x.tolist() for x in got] == [[-1] * 3, [0] * 3, [0], [], [1]]
    # positions past 2^31 - 1 are limited, and no page is asked for
    got = ga.kv4_append(_i32([[1]]), _i32([2 ** 31 - 2]), _i32([5]), _i32([3]), _i32([1]), 16, 5)
    assert got.slots.tolist() == [-1] * 5 and got.lengths.tolist() == [2 ** 31 - 1] and got.free_count.tolist() == [1]


def test_append_slots_past_32_bits():
    from grinqh import attention as ga
    got = ga.kv4_append(_i32([[-1, -1]]), _i32([0]), _i32([20]), _i32([4, 2 ** 31 - 1]), _i32([2]), 32, 20)
    assert got.slots.tolist() == [(2 ** 31 - 1) * 32 + i for i in range(20)]


# ---------------------------------------------------------------- summaries

def _codes(x):
    """8-bit codes along the last axis and their step, fp64"""
    top = np.abs(x).max(-1, keepdims=True)
    exponent = np.frexp(np.where(top > 0, top, 1.0))[1] - 1
    step = np.where(top > 0, np.ldexp(1.0, exponent - 6), 0.0)
    return np.clip(np.rint(x / np.where(step > 0, step, 1.0)), -127, 127).astype(np.int8), step


def _summary_ref(keys, lens, group, page):
    """per sequence: codes int8 and steps [pages, heads, .] of its pages, of keys [T, H, D] as the cache keeps them"""
    out = []
    for k, n in zip(keys, lens):
        kf = k.float().cpu().numpy()
        c, s, m = _quantize(kf, group)
        wide = lambda a: np.repeat(a.astype(np.float64), group, -1)  # noqa: E731
        kept = (wide(m) + wide(s) * c)[:n]
        means = np.stack([kept[i:i + page].sum(0) / len(kept[i:i + page]) for i in range(0, n, page)])
        out.append(_codes(np.where(np.isfinite(means), means, 0.0)))
    return out


def _steps(summary, d):
    return np.ascontiguousarray(summary[..., d:d + 4]).view(np.float32)


@pytest.mark.parametrize("dtype,d,group,page,heads", LAYOUTS)
@pytest.mark.parametrize("seqs", [1, 70])
def test_summarize(dtype, d, group, page, heads, seqs):
    from grinqh import attention as ga
    rng = np.random.default_rng(d + group + seqs)
    lens = [333] if seqs == 1 else rng.integers(0, 100, seqs).tolist()
    cache, table, lengths, kv = _paged(rng, lens, heads, d, page, group, dtype)
    summary = ga.kv4_summary(cache)
    before = torch.randint(-128, 128, summary.shape, dtype=torch.int8, device="cuda")
    summary.copy_(before)
    starts = [n // 2 for n in lens]
    ga.kv4_summarize(cache, summary, table, _i32(starts), lengths)
    got, old, tab = summary.cpu().numpy(), before.cpu().numpy(), table.cpu().numpy()
    want = _summary_ref([k for k, _ in kv], lens, group, page) if seqs == 1 else None
    for i, n in enumerate(lens):
        if n == 0:
            continue
        codes, steps = want[0] if seqs == 1 else _summary_ref([kv[i][0]], [n], group, page)[0]
        for j in range(starts[i] // page, -(-n // page)):
            at = tab[i, j]
            assert np.array_equal(got[at, :, :d], codes[j]), (i, j)
            assert np.array_equal(_steps(got[at], d), steps[j].astype(np.float32)), (i, j)
            old[at, :, :d + 4] = got[at, :, :d + 4]
    assert np.array_equal(got, old)  # nothing else is written


def test_summarize_special_keys():
    """zeros, constants, limits, tiny keys, NaN (counted as 0), what stands behind the last token"""
    from grinqh import attention as ga
    rng = np.random.default_rng(4)
    page, n = 16, 6 * 16 + 5
    k = rng.standard_normal((n, 2, 128)).astype(np.float32)
    k[:16], k[16:32], k[32:48] = 0.0, -1.75, np.where(np.arange(128) % 2, LIMIT, -LIMIT)
    k[48:64] *= 6e-8
    k[64 + 3, 1, 5] = np.nan
    kt = torch.from_numpy(k).half().cuda()
    cache = ga.kv4_cache(9, 2, 128, page, 32)
    cache.fill_(0xFF)
    table = _i32([[3, 1, 4, 8, 5, 0, 2]])
    at = torch.arange(n).cuda()
    ga.kv4_store(cache, kt, kt, table[0, at // 16].long() * 16 + at % 16)
    summary = ga.kv4_summary(cache)
    ga.kv4_summarize(cache, summary, table, _i32([0]), _i32([n]))
    codes, steps = _summary_ref([kt], [n], 32, page)[0]
    got = summary[table[0].long()].cpu().numpy()
    assert np.array_equal(got[:, :, :128], codes) and np.array_equal(_steps(got, 128), steps.astype(np.float32))
    assert not codes[4, 1, :32].any() and codes[4, 1, 32:].any()


def test_summarize_passes_over_what_is_not_there():
    """empty ranges, starts past the end, pages outside the cache, lengths past the table, no sequences"""
    from grinqh import attention as ga
    cache = ga.kv4_cache(4, 1, 64)
    k = torch.ones((64, 1, 64), dtype=torch.float16, device="cuda")
    ga.kv4_store(cache, k, k, torch.arange(64).cuda())
    for table, starts, lengths, touched in (
            ([[0, 1], [2, 3]], [5, 40], [5, 20], []), ([[0, 1], [2, 3]], [16, -3], [17, 1], [1, 2]),
            ([[-1, 1], [9, 2 ** 31 - 1]], [0, 0], [32, 32], [1]), ([[0, 1], [2, 3]], [0, 31], [99, 2 ** 31 - 1], [0, 1, 3]),
            ([[0, 1], [2, 3]], [0, 100], [-5, 200], [])):
        summary = ga.kv4_summary(cache)
        ga.kv4_summarize(cache, summary, _i32(table), _i32(starts), _i32(lengths))
        assert summary.ne(0).any(-1).any(-1).nonzero().flatten().tolist() == touched
    ga.kv4_summarize(cache, summary, _i32([[0]])[:0], _i32([]), _i32([]))


# ---------------------------------------------------------------- selection

def _select_ref(q, summary, table, lengths, page, count):
    """numpy: q [B, H, D] fp64, summary int8 [pages, KV, D + 16]; indices [B, KV, count], lengths"""
    b, hq, d = q.shape
    pages, hkv, _ = summary.shape
    capacity = table.shape[1] * page
    out, after = np.full((b, hkv, count), -1, np.int32), []
    q = np.clip(np.nan_to_num(q, nan=0.0, posinf=np.inf, neginf=-np.inf), -3.4028234663852886e38, 3.4028234663852886e38)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), capacity)
        held = -(-n // page)
        after.append(2 ** 31 - 1 if lengths[i] > capacity else n - max(held - count, 0) * page)
        for h in range(hkv):
            places = list(range(held))
            if held > count:
                codes, steps = _codes(q[i].reshape(hkv, -1, d)[h])
                factor = np.maximum(steps / (steps.max() if steps.max() > 0 else 1.0), 2.0 ** -40)
                at = table[i, :held]
                bad = (at < 0) | (at >= pages)
                rec = summary[np.where(bad, 0, at), h]
                score = ((codes.astype(np.float64) @ rec[:, :d].T.astype(np.float64)) * factor).max(0)
                score = np.where(bad, np.inf, score * _steps(rec, d)[:, 0].astype(np.float64))
                middle = sorted(range(1, held - 1), key=lambda j: (-score[j], j))[:count - 2]
                places = [0] + sorted(middle) + [held - 1]
            out[i, h, :len(places)] = table[i, places]
    return out, after


def _random_summary(rng, pages, heads, d, spread=3):
    s = rng.integers(-127, 128, (pages, heads, d + 16)).astype(np.int8)
    s[..., d:d + 4] = np.ldexp(1.0, rng.integers(-6, -6 + spread, (pages, heads, 1))).astype(np.float32).view(np.int8)
    return s


def _check_select(rng, q, summary, table, lengths, page, count):
    from grinqh import attention as ga
    got, after = ga.kv4_select(q, torch.from_numpy(summary).cuda(), _i32(table), _i32(lengths), page, count)
    want, want_after = _select_ref(q.double().cpu().numpy(), summary, np.asarray(table), lengths, page, count)
    assert after.tolist() == want_after
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128), ("f16", 128), ("bf16", 256)])
@pytest.mark.parametrize("hkv,per", [(2, 4), (1, 1), (3, 5), (1, 16), (2, 17), (1, 40)])
def test_select(dtype, d, hkv, per):
    rng = np.random.default_rng(d + per)
    lens = [0, 1, 16, 17, 33, 32 * 16, 700, 1000, 999, 48]
    pages, width = 900, 64
    summary = _random_summary(rng, pages, hkv, d)
    table = rng.permutation(pages)[:len(lens) * width].reshape(len(lens), width)
    for count in (2, 3, 20, 62, 63, 64, 100):
        q = _randn(rng, len(lens), hkv * per, d, dtype=dtype)
        _check_select(rng, q, summary, table, lens, 16, count)


@pytest.mark.parametrize("width", [2047, 2048, 2049, 4100, 8192, 8193, 20000])
@pytest.mark.parametrize("count", [2, 3, 129, 1500])
def test_select_wide_tables(width, count):
    """both launches, scores in registers and read again"""
    rng = np.random.default_rng(width)
    summary = _random_summary(rng, width + 50, 2, 64)
    table = np.stack([rng.permutation(width + 50)[:width] for _ in range(3)])
    q = _randn(rng, 3, 8, 64)
    _check_select(rng, q, summary, table, [width * 16 - 3, width * 16, width * 8], 16, count)


@pytest.mark.parametrize("width", [300, 3000, 9000])
def test_select_equal_scores(width):
    """ties go to the page that comes first: pages all alike, half of them, zeros, one far from the rest"""
    rng = np.random.default_rng(5)
    base = _random_summary(rng, width, 1, 64, spread=1)
    q = _randn(rng, 1, 4, 64)
    table = rng.permutation(width).reshape(1, -1)
    alike = np.repeat(base[:1], width, 0)
    half = alike.copy()
    half[::2] = base[::2]
    zeros = np.zeros_like(base)
    far = alike.copy()
    far[table[0, width // 2], 0, 64:68] = np.float32(2.0 ** 60).reshape(1).view(np.int8)
    few = base.copy()
    few[:, 0, :64] = rng.integers(0, 2, (width, 1)).astype(np.int8)  # two different scores
    for summary in (alike, half, zeros, far, few):
        for count in (2, 3, 77, width - 1):
            _check_select(rng, q, summary, table, [width * 16], 16, count)


def test_select_special_queries_and_pages():
    """zeros, NaN, infinities, heads of very different size; bad pages score highest; a length past the table stays one"""
    rng = np.random.default_rng(6)
    summary = _random_summary(rng, 200, 2, 128)
    table = rng.permutation(200)[:180].reshape(3, 60)
    q = _randn(rng, 3, 8, 128, dtype="bf16")
    q[0, :4] = 0
    q[0, 5, 7], q[1, 2, 3], q[1, 6, 0] = float("nan"), float("inf"), float("-inf")
    q[2, 0] *= 1e30
    q[2, 1] *= 1e-30
    q[2, 5] *= 1e-38
    table = table.copy()
    table[1, 7], table[1, 20], table[2, 3] = -1, 200, 2 ** 31 - 1
    for count in (2, 3, 4, 30):
        _check_select(rng, q, summary, table, [960, 955, 961], 16, count)


def test_select_leaves_attention_to_show_bad_pages():
    from grinqh import attention as ga
    rng = np.random.default_rng(7)
    cache, table, lengths, kv = _paged(rng, [500, 500], 2, 64, 16, 64, "f16")
    summary = ga.kv4_summary(cache)
    ga.kv4_summarize(cache, summary, table, torch.zeros_like(lengths), lengths)
    q = _randn(rng, 2, 8, 64)
    table[1, 9] = -1
    pages, some = ga.kv4_select(q, summary, table, lengths, 16, 5)
    out = ga.kv4_attention(q, cache, pages, some)
    assert bool(out[1].isnan().all()) and not bool(out[0].isnan().any())
    pages, some = ga.kv4_select(q, summary, table, lengths + 100, 16, 5)
    assert bool(ga.kv4_attention(q, cache, pages, some).isnan().all())


# ---------------------------------------------------------------- attention over a page table per head

@pytest.mark.parametrize("dtype,d,group,page,hkv", LAYOUTS)
@pytest.mark.parametrize("per", [1, 4, 17])
def test_attention_over_selected_pages(dtype, d, group, page, hkv, per):
    """every head its own pages, in its own order"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d + group + per)
    lens = [0, 5, 16 * page, 7 * page + 3, 9 * page]
    cache, table, lengths, kv = _paged(rng, lens, hkv, d, page, group, dtype)
    q = _randn(rng, len(lens), hkv * per, d, dtype=dtype)
    tab = table.cpu().numpy()
    width, some = 6, []
    pages = np.full((len(lens), hkv, width), -1, np.int32)
    picked = [[None] * hkv for _ in lens]
    for i, n in enumerate(lens):
        held = -(-n // page)
        take = min(held, width)
        some.append(n - (held - take) * page)
        for h in range(hkv):
            places = np.sort(rng.permutation(max(held - 1, 0))[:max(take - 1, 0)]).tolist() + [held - 1] * (held > 0)
            pages[i, h, :take] = tab[i, places]
            picked[i][h] = np.concatenate([np.arange(j * page, min((j + 1) * page, n)) for j in places] + [np.arange(0)])
    tables = torch.from_numpy(pages).cuda()
    # as one table, and as slices of a larger one whose rows lie apart
    apart = torch.full((len(lens), hkv + 1, 2 * width), -9, dtype=torch.int32, device="cuda")
    apart[:, 1:, 3:3 + width] = tables
    out = ga.kv4_attention(q, cache, tables, _i32(some))
    assert torch.equal(out, ga.kv4_attention(q, cache, apart[:, 1:, 3:3 + width], _i32(some)))
    for h in range(hkv):
        seqs = [tuple(x[torch.from_numpy(picked[i][h].astype(np.int64)).cuda(), h:h + 1] for x in kv[i])
                for i in range(len(lens))]
        _check_decode(out[:, h * per:(h + 1) * per], q[:, h * per:(h + 1) * per], seqs, group, dtype)


def test_attention_over_one_table_for_all_heads():
    """the same pages for every head, given per head: nothing changes"""
    from grinqh import attention as ga
    rng = np.random.default_rng(1)
    cache, table, lengths, kv = _paged(rng, [3000, 17, 400], 4, 128, 16, 64, "f16")
    q = _randn(rng, 3, 16, 128)
    want = ga.kv4_attention(q, cache, table, lengths)
    assert torch.equal(ga.kv4_attention(q, cache, table.unsqueeze(1).expand(-1, 4, -1), lengths), want)
    assert torch.equal(ga.kv4_attention(q, cache, table.unsqueeze(1).repeat(1, 4, 1), lengths), want)


# ---------------------------------------------------------------- together

class _Server:
    """A few sequences served as a program would: room, store, summaries, attention."""

    def __init__(self, rng, seqs, hkv=2, per=4, d=128, page=16, group=32, pages=200, width=40, dtype="f16"):
        from grinqh import attention as ga
        self.ga, self.page, self.dtype, self.group = ga, page, dtype, group
        self.cache = ga.kv4_cache(pages, hkv, d, page, group)
        self.cache.fill_(0xFF)
        self.summary = ga.kv4_summary(self.cache)
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.free = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda()
        self.free_count = _i32([pages])

    def step(self, q, k, v, counts, count=None):
        """q, k, v: buffers of some rows, the new tokens in front"""
        ga = self.ga
        r = ga.kv4_append(self.table, self.lengths, counts, self.free, self.free_count, self.page, q.shape[0])
        ga.kv4_store(self.cache, k, v, r.slots)
        ga.kv4_summarize(self.cache, self.summary, self.table, self.lengths, r.lengths)
        self.lengths.copy_(r.lengths)
        self.free_count.copy_(r.free_count)
        if count is None:
            return ga.kv4_chunk_attention(q, self.cache, self.table, self.lengths, r.ends)
        pages, some = ga.kv4_select(q, self.summary, self.table, self.lengths, self.page, count)
        return ga.kv4_attention(q, self.cache, pages, some)


def test_serving_steps_together():
    """prompts in chunks, drafted tokens, single tokens over all pages and over selected ones"""
    rng = np.random.default_rng(3)
    s = _Server(rng, 3)
    held = [(torch.zeros((0, 2, 128), dtype=torch.float16, device="cuda"),) * 2 for _ in range(3)]
    for news in ([100, 0, 30], [0, 64, 7], [1, 1, 1], [4, 3, 4], [200, 1, 1], [1, 1, 1]):
        rows = sum(news) + 6
        q, k, v = _randn(rng, rows, 8, 128), _randn(rng, rows, 2, 128), _randn(rng, rows, 2, 128)
        out = s.step(q, k, v, _i32(news))
        at = 0
        for i, n in enumerate(news):
            held[i] = tuple(torch.cat((a, b[at:at + n])) for a, b in zip(held[i], (k, v)))
            at += n
        assert s.lengths.tolist() == [x.shape[0] for x, _ in held]
        _check_chunk(out, q, held, news, 32, "f16")
    used = s.table[s.table >= 0].tolist()
    assert len(set(used)) == len(used) and len(used) + int(s.free_count) == 200
    # all pages selected: the same as the attention over all of them
    q, k, v = _randn(rng, 3, 8, 128), _randn(rng, 3, 2, 128), _randn(rng, 3, 2, 128)
    out = s.step(q, k, v, _i32([1, 1, 1]), count=40)
    held = [tuple(torch.cat((a, b[i:i + 1])) for a, b in zip(held[i], (k, v))) for i in range(3)]
    _check_decode(out, q, held, 32, "f16")
    # a needle: the page with the query's own direction is among the selected ones
    pages, some = s.ga.kv4_select(held[0][0][150].repeat_interleave(4, 0).unsqueeze(0) * 4, s.summary, s.table[:1],
                                  s.lengths[:1], 16, 4)
    assert all(int(s.table[0, 150 // 16]) in row for row in pages[0].tolist())
    # the summary that grew with the steps is the one that is made at once
    again = s.ga.kv4_summary(s.cache)
    s.ga.kv4_summarize(s.cache, again, s.table, torch.zeros_like(s.lengths), s.lengths)
    pick = torch.tensor(s.table[s.table >= 0].tolist()).cuda()
    assert torch.equal(again[pick][..., :132], s.summary[pick][..., :132])


@pytest.mark.parametrize("rows,count", [(3, None), (9, None), (40, None), (3, 6)])
def test_captured_steps(rows, count):
    """Two captured graphs of whole steps, replayed in turn and at the same time on two streams, with eager work
    between: each equals the eager program."""
    rng = np.random.default_rng(rows)
    news = {3: [1, 1, 1], 9: [3, 3, 3], 40: [1, 38, 1]}[rows]
    q, k, v = _randn(rng, rows, 8, 128), _randn(rng, rows, 2, 128), _randn(rng, rows, 2, 128)
    counts = _i32(news)
    start = _i32([500, 30, 120])

    def server(seed):
        g = np.random.default_rng(seed)
        s = _Server(g, 3, width=50)
        kk, vv = _randn(g, 700, 2, 128), _randn(g, 700, 2, 128)
        s.step(_randn(g, 700, 8, 128), kk, vv, start)
        return s

    eager = [server(i) for i in (1, 2)]
    captured = [server(i) for i in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the workspaces of the capturing stream
        server(3).step(q, k, v, counts, count)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(s.step(q, k, v, counts, count))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        if turn % 2:
            torch.cuda.synchronize()
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            torch.cuda.synchronize()
        else:
            for graph in graphs:
                graph.replay()
                torch.randn(1000, device="cuda").sum()
        for s, c, out in zip(eager, captured, outs):
            want = s.step(q, k, v, counts, count)
            assert torch.equal(c.lengths, s.lengths) and torch.equal(c.table, s.table)
            assert torch.equal(out, want), turn
