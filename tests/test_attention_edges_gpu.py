"""GPU tests of the attention operators at the edges of their inputs: values
and rows that must not count, layouts of memory, extreme magnitudes, runs
joined over many blocks.  The oracles and bounds are those of
test_attention_gpu.py; where two calls must agree, they agree bit for bit."""
import numpy as np
import pytest
import torch

from test_attention_gpu import DT, LIMIT, _check_decode, _check_prompt, _dev, _ends, _paged, _params, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


# ---------------------------------------------------------------- values that a row must not see

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [(300, 300), (70, 333), (290, 200), (1, 65), (20, 20)])
def test_prompt_later_values_do_not_count(dtype, d, rows, keys):
    """NaN and infinities in values: in the channels of the rows that see them, as the sum gives them, and nowhere
    else, whatever tile the rows share with them"""
    from grinqh import attention as ga
    rng = np.random.default_rng(rows + keys + d)
    hq, hkv = 4, 2
    ends, key_ends = [0, 17, 17 + rows], [0, 30, 30 + keys]
    q = _randn(rng, ends[-1], hq, d, dtype=dtype)
    k, v = (_randn(rng, key_ends[-1], hkv, d, dtype=dtype) for _ in (0, 1))
    nan, inf = float("nan"), float("inf")
    spots = [(0, 0, 3, nan), (1, 1, 4, inf), (5, 0, 9, -inf), (40, 1, 63, nan), (63, 0, 20, inf), (64, 0, 21, -inf),
             (64, 1, 21, inf), (100, 1, 21, -inf), (127, 0, 8, nan), (128, 1, 5, inf), (150, 0, 8, inf),
             (199, 0, 33, nan), (keys - 1, 0, 2, nan), (keys - 1, 1, 1, inf), (keys - 2, 1, 62, -inf)]
    spots = [s for s in spots if 0 <= s[0] < keys]
    bad, none = v.clone(), v.clone()
    effect = torch.zeros_like(q, dtype=torch.float32)
    row = torch.arange(rows, device="cuda")
    for key, head, channel, value in spots:
        bad[30 + key, head, channel] = value
        none[30 + key, head, channel] = 0.0
        seen = torch.where(row + keys - rows >= key, value, 0.0).view(-1, 1)
        effect[17:, 2 * head:2 * head + 2, channel] += seen
    out = ga.prompt_attention(q, k, bad, _dev(ends), _dev(key_ends))
    want = ga.prompt_attention(q, k, none, _dev(ends), _dev(key_ends)) + effect.to(q.dtype)
    assert bool(want.isfinite().any())
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(0.0, inf, -inf), want.nan_to_num(0.0, inf, -inf))


def test_prompt_infinite_values_of_small_weight():
    """an infinite value counts for the rows that see it also where its weight rounds to zero in fp16"""
    from grinqh import attention as ga
    rng = np.random.default_rng(77)
    n, key, inf = 400, 150, float("inf")
    q, k = (torch.zeros((n, 2, 128), dtype=torch.float16, device="cuda") for _ in (0, 1))
    q[:, :, 0], k[:, :, 0], k[0, :, 0] = 16.0, -20.0, 0.0  # exp(-20) and the first key
    v = _randn(rng, n, 2, 128)
    want = ga.prompt_attention(q, k, v, _dev([0, n]), scale=1.0 / 16)
    v[key, 0, 3], v[key, 1, 7], v[key + 100, 1, 7] = inf, inf, -inf
    out = ga.prompt_attention(q, k, v, _dev([0, n]), scale=1.0 / 16)
    want[key:, 0, 3], want[key:key + 100, 1, 7] = inf, inf
    assert bool(out[key + 100:, 1, 7].isnan().all())
    out[key + 100:, 1, 7] = want[key + 100:, 1, 7] = 0.0
    assert torch.equal(out, want)


# ---------------------------------------------------------------- rows of no sequence

@pytest.mark.parametrize("ends", [[9, 40, 70], [300, 300, 333], [77], [200, 201], [1, 80, 80]])
@pytest.mark.parametrize("heads", [4, 8])
def test_prompt_rows_before_the_first_sequence(ends, heads):
    """rows in front of the first sequence give zeros, as those behind the last do"""
    from grinqh import attention as ga
    rng = np.random.default_rng(ends[0])
    tokens = ends[-1] + 50
    q, k, v = (_randn(rng, tokens, n, 64) for n in (heads, 2, 2))
    stale = torch.full((tokens, heads, 64), float("nan"), dtype=q.dtype, device="cuda")
    del stale  # the result is likely to lie where this was
    out = ga.prompt_attention(q, k, v, _dev(ends))
    _check_prompt(out, q, k, v, ends, ends, "f16")
    key_ends = [e - ends[0] for e in ends]
    stale = torch.full((tokens, heads, 64), float("nan"), dtype=q.dtype, device="cuda")
    del stale, out
    _check_prompt(ga.prompt_attention(q, k, v, _dev(ends), _dev(key_ends)), q, k, v, ends, key_ends, "f16")


# ---------------------------------------------------------------- layouts that the kernels cannot read in place

def _odd_layouts(x):
    """x [tokens, heads, d] where its rows are not 16-byte aligned although torch calls the tensor contiguous, and
    one token or head with distances that do not matter"""
    t, h, d = x.shape
    shifted = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(t, h, d)
    yield shifted.copy_(x)
    if t == 1:
        wide = torch.empty((4, h, d), dtype=x.dtype, device=x.device)
        wide[:1] = x
        for distance in (0, 3, (1 << 23) + 8):
            yield wide.as_strided((1, h, d), (distance, d, 1))
    if h == 1:
        wide = torch.empty((t, 1, d + 1), dtype=x.dtype, device=x.device)
        yield wide[:, :, 1:].copy_(x)
        yield x.as_strided((t, 1, d), (d, 5, 1))


@pytest.mark.parametrize("tokens", [1, 2, 33])
@pytest.mark.parametrize("heads", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_layouts_are_copied(tokens, heads, d):
    from grinqh import attention as ga
    rng = np.random.default_rng(tokens)
    q, k, v = (_randn(rng, tokens, heads, d) for _ in range(3))
    slots = torch.arange(tokens).cuda()
    table = torch.zeros((tokens, 3), dtype=torch.int32, device="cuda")
    table[:, 1], table[:, 2] = 1, 2
    lengths = torch.full((tokens,), tokens, dtype=torch.int32, device="cuda")
    ends = _dev([0, tokens])
    cache, again = ga.kv4_cache(3, heads, d), ga.kv4_cache(3, heads, d)
    ga.kv4_store(cache, k, v, slots)
    decode, prompt = ga.kv4_attention(q, cache, table, lengths), ga.prompt_attention(q, k, v, ends)
    for k2, v2, q2 in zip(_odd_layouts(k), _odd_layouts(v), _odd_layouts(q)):
        for a, b in ((k2, v), (k, v2)):
            again.zero_()
            ga.kv4_store(again, a, b, slots)
            assert torch.equal(again, cache)
        assert torch.equal(ga.kv4_attention(q2, cache, table, lengths), decode)
        for args in ((q2, k, v), (q, k2, v), (q, k, v2)):
            assert torch.equal(ga.prompt_attention(*args, ends), prompt)


# ---------------------------------------------------------------- workspaces

def test_largest_batch_covers_smaller_ones_in_a_capture():
    """a batch too large to share its sequences, run once, leaves the workspace that smaller batches share theirs in"""
    from grinqh import attention as ga
    rng = np.random.default_rng(21)
    cache, table, lengths, kv = _paged(rng, [3000, 40], 1, 64, 16, 64, "f16")
    pick = torch.arange(1025).cuda() % 2
    q = _randn(rng, 2, 2, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ga.kv4_attention(q[pick], cache, table[pick], lengths[pick])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ga.kv4_attention(q, cache, table, lengths)
    torch.cuda.synchronize()
    for i in range(3):
        q.copy_(_randn(rng, 2, 2, 64))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        _check_decode(got, q, kv, 64, "f16")
        assert torch.equal(got, ga.kv4_attention(q, cache, table, lengths))


# ---------------------------------------------------------------- magnitudes

def test_values_at_the_limit_stay_finite():
    """a scale that rounds up makes the largest code stand for more than fp16 holds: results are limited as the stored
    values are; NaN stays NaN"""
    from grinqh import attention as ga
    d = 128
    x = torch.zeros((6, 1, d), dtype=torch.float16, device="cuda")
    x[0, 0, ::2] = LIMIT                                  # scale 4368: code 15 stands for 65520
    x[1, 0, ::2], x[1, 0, 1::2] = LIMIT, -LIMIT           # scale 8736: code 15 stands for 65536
    x[2, 0, 3] = float("inf")
    x[3, 0, 5] = float("-inf")
    x[4], x[5, 0, 7] = -LIMIT, float("nan")
    slots = torch.arange(6).cuda()
    cache = ga.kv4_cache(6, 1, d, 16, 32)
    ga.kv4_store(cache, x, x, slots * 16)
    k, v = ga.kv4_load(cache, slots * 16, torch.float16)
    for got in (k, v):
        assert bool(got[:5].isfinite().all()) and float(got[0].max()) == LIMIT and float(got[1].max()) == LIMIT
        assert float(got[2].max()) == LIMIT and float(got[3].min()) == -LIMIT and bool((got[4] == -LIMIT).all())
        assert bool(got[5, 0, :32].isnan().all())
    wide, _ = ga.kv4_load(cache, slots * 16, torch.bfloat16)
    assert float(wide[0].max()) == 65536.0  # the limit, and 65520, to 8 bits
    # one key each
    lengths = torch.ones(6, dtype=torch.int32, device="cuda")
    q = torch.ones((6, 1, d), dtype=torch.float16, device="cuda")
    out = ga.kv4_attention(q, cache, slots.int().view(6, 1), lengths)
    assert bool(out[:5].isfinite().all()) and bool(out[5].isnan().all())
    # a weight's rounding (2^-11) times what is left of 15 codes about their middle, and the result's own rounding
    scale = torch.tensor([4368.0, 8736.0, 4368.0, 4368.0, 0.0], device="cuda").view(5, 1, 1)
    assert bool(((out[:5].float() - v[:5].float()).abs() <= 2.0 ** -11 * (7.5 * scale + v[:5].float().abs())).all())
    # many equal keys, joined over several blocks
    cache = ga.kv4_cache(200, 1, d, 16)
    t = torch.arange(3000).cuda()
    ga.kv4_store(cache, x[:1].expand(3000, -1, -1), x[1:2].expand(3000, -1, -1), t)
    q = torch.ones((1, 2, d), dtype=torch.float16, device="cuda")
    out = ga.kv4_attention(q, cache, torch.arange(200).int().cuda().view(1, -1), torch.tensor([3000]).int().cuda())
    assert bool(out.isfinite().all()) and bool((out.float().abs() >= LIMIT * (1 - 2.0 ** -9)).all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_values_at_the_limit_stay_finite(d):
    """fp16 weights are rounded and their sum is not, so that a mean of values at the limit may come out above it: one
    key of the second tile has nearly all the weight, which is not a power of two as the reference is the first key's"""
    from grinqh import attention as ga
    n, key = 400, 70
    q, k = (torch.zeros((n, 2, d), dtype=torch.float16, device="cuda") for _ in (0, 1))
    q[:, :, 0] = 16.0
    q[:, :, 1] = torch.linspace(3.0, 5.4, n).cuda().half().view(n, 1)
    k[:, :, 0] = -20.0
    k[0, :, 0], k[key, :, 0], k[key, :, 1] = 0.0, 0.0, 16.0
    v = torch.full((n, 2, d), LIMIT, dtype=torch.float16, device="cuda")
    v[:, :, 1::2] = -LIMIT
    out = ga.prompt_attention(q, k, v, _dev([0, n]), scale=1.0 / 16)
    assert bool(out.isfinite().all())
    _check_prompt(out, q, k, v, [0, n], [0, n], "f16", 1.0 / 16)
    seen, inf = 150, float("inf")  # infinities are no such excess
    v[seen, 1, 2], v[seen, 1, 3], v[key, 0, 5] = inf, -inf, -inf
    again = ga.prompt_attention(q, k, v, _dev([0, n]), scale=1.0 / 16)
    out[seen:, 1, 2], out[seen:, 1, 3], out[key:, 0, 5] = inf, -inf, -inf
    assert torch.equal(again, out)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_far_negative_logits(d):
    """logits of -10^33 and below, all a row has: the largest takes the weight"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    n = 150
    q = torch.full((n, 2, d), 2.0 ** 56, dtype=torch.bfloat16, device="cuda")
    k = (-2.0 ** 50 * torch.arange(100, 100 + n).cuda()).view(n, 1, 1).expand(n, 1, d).bfloat16()  # 8 bits each
    v = _randn(rng, n, 1, d, dtype="bf16")
    out = ga.prompt_attention(q, k, v, _dev([0, n]))
    assert torch.equal(out, v[:1].expand(n, 2, d))
    out = ga.prompt_attention(-q, k, v, _dev([0, n]))
    assert torch.equal(out, v.expand(n, 2, d))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_large_logits_of_few_bits(d, dtype):
    """logits around +-2^30, where fp32 steps by 64: they are sums of 16-bit integers' products here, exact in fp32, and
    tell keys apart by more than that, so that the largest key, or several equal ones, takes all weight"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    n = 300
    size = 2.0 ** 14
    k = torch.zeros((n, 2, d), device="cuda")
    steps = torch.from_numpy(rng.permutation(np.repeat(np.arange(n // 2), 2))).cuda().float()
    k[:, 0, 0] = size * (64 + steps % 64)
    k[:, 1, 1] = -size * (64 + steps % 64)
    k = (k / 64).to(DT[dtype])
    q = torch.full((n, 4, d), size, dtype=DT[dtype], device="cuda")
    v = _randn(rng, n, 2, d, dtype=dtype)
    _check_prompt(ga.prompt_attention(q, k, v, _dev([0, n]), scale=1.3), q, k, v, [0, n], [0, n], dtype, 1.3)


@pytest.mark.parametrize("tokens", [5, 40, 3000])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_far_logits(tokens, d):
    """logits of -10^33 and 10^34: the largest, or all that bf16 rounds to it, take the weight"""
    from grinqh import attention as ga
    rng = np.random.default_rng(tokens + d)
    cache = ga.kv4_cache(190, 1, d)
    t = torch.arange(tokens).cuda()
    k = torch.linspace(100.0, 1000.0, tokens).cuda().view(-1, 1, 1).expand(tokens, 1, d).bfloat16()
    v = _randn(rng, tokens, 1, d, dtype="bf16")
    ga.kv4_store(cache, k, v, t)
    _, kept = ga.kv4_load(cache, t, torch.bfloat16)
    table, lengths = torch.arange(190).int().cuda().view(1, -1), torch.tensor([tokens]).int().cuda()
    q = torch.full((1, 2, d), 1e31, dtype=torch.bfloat16, device="cuda")
    for sign, same in ((-1.0, k[:, 0, 0] == k[0, 0, 0]), (1.0, k[:, 0, 0] == k[-1, 0, 0])):
        out = ga.kv4_attention(sign * q, cache, table, lengths)
        want = kept[same].double()
        # a weight's rounding times the codes about their middle; two roundings to bf16
        step = (want.amax(-1) - want.amin(-1)).max() / 15
        tol = 2.0 ** -11 * 7.5 * step + 2.0 ** -7 * want.abs().mean(0)
        assert bool(((out.double() - want.mean(0)).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [40, 3000])
def test_decode_large_logits_of_few_bits(tokens, dtype):
    """logits around +-2^36, exact in fp32 (codes 0 to 15 of one scale, a power of two), that tell tokens apart by more
    than fp32's step there"""
    from grinqh import attention as ga
    rng = np.random.default_rng(tokens)
    d, sign = 64, torch.tensor([1.0, -1.0], device="cuda")
    code = torch.from_numpy(rng.integers(0, 16, tokens)).cuda()
    k = torch.zeros((tokens, 1, d), device="cuda")
    k[:, :, 0::2], k[:, :, 1::2] = 30720.0, 0.0  # 15 * 2048
    k[:, 0, 0] = code * 2048.0
    k, v = k.to(DT[dtype]), _randn(rng, tokens, 1, d, dtype=dtype)
    cache = ga.kv4_cache(190, 1, d)
    t = torch.arange(tokens).cuda()
    ga.kv4_store(cache, k, v, t)
    _, kept = ga.kv4_load(cache, t, torch.bfloat16)
    q = torch.zeros((1, 2, d), dtype=DT[dtype], device="cuda")
    q[0, :, 0] = sign.to(q.dtype) * 2.0 ** 14
    q[0, :, 2] = 3 * 2.0 ** 14
    out = ga.kv4_attention(q, cache, torch.arange(190).int().cuda().view(1, -1), torch.tensor([tokens]).int().cuda(),
                           scale=1.3)
    for head, best in ((0, code.max()), (1, code.min())):
        want = kept[code == best].double().mean(0)[0]
        assert float((out[0, head].double() - want).abs().max()) <= 2.0 ** -7 * float(kept.abs().max())


@pytest.mark.parametrize("tokens", [5, 40, 3000])
@pytest.mark.parametrize("size,scale", [(2.0 ** 120, None), (1e-25, 1e-25), (2.0 ** 127, 1e3), (1e-38, 1e-37)])
def test_decode_queries_of_any_size(tokens, size, scale):
    """queries and scales whose product with the codes' unit leaves fp32's range, equal logits: the mean of all values"""
    from grinqh import attention as ga
    rng = np.random.default_rng(tokens)
    d = 128
    cache = ga.kv4_cache(190, 1, d)
    t = torch.arange(tokens).cuda()
    v = _randn(rng, tokens, 1, d, dtype="bf16")
    ga.kv4_store(cache, torch.zeros_like(v), v, t)
    _, kept = ga.kv4_load(cache, t, torch.bfloat16)
    table, lengths = torch.arange(190).int().cuda().view(1, -1), torch.tensor([tokens]).int().cuda()
    q = torch.full((1, 2, d), size, dtype=torch.bfloat16, device="cuda")
    out = ga.kv4_attention(q, cache, table, lengths, scale=scale)
    assert float((out.double() - kept.double().mean(0)).abs().max()) <= 2.0 ** -7 * float(kept.abs().max())


# ---------------------------------------------------------------- refusals

def test_refuses_caches_without_heads():
    from grinqh import attention as ga
    cache = torch.zeros((2, 0, 1, 2176), dtype=torch.uint8, device="cuda")
    q = torch.ones((1, 4, 128), dtype=torch.float16, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for call in (lambda: ga.kv4_attention(q, cache, one.view(1, 1), one), lambda: ga.kv4_load(cache, one.long()),
                 lambda: ga.kv4_store(cache, q[:, :0], q[:, :0], one.long())):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- sequences shared by many blocks

@pytest.mark.parametrize("d,per", [(64, 3), (64, 16), (128, 5), (128, 7), (128, 16), (256, 1), (256, 3), (256, 7),
                                   (256, 12), (256, 16), (256, 17)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_join(d, per, dtype):
    """runs joined where the columns of a run are fewer than a block's threads, do not divide them, or exceed them"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d + per)
    lens = [5000, 33, 2049]
    cache, table, lengths, kv = _paged(rng, lens, 1, d, 32, 64, dtype)
    q = _randn(rng, len(lens), per, d, dtype=dtype)
    for _ in range(2):  # the counters are zero again after a call
        _check_decode(ga.kv4_attention(q, cache, table, lengths), q, kv, 64, dtype)


@pytest.mark.parametrize("d,per", [(64, 2), (128, 5), (256, 16)])
def test_decode_join_many_runs(d, per):
    """more than 64 runs of one sequence, and more than one round of loads of them"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    cache, table, lengths, kv = _paged(rng, [75001], 1, d, 64, d, "f16")
    q = _randn(rng, 1, per, d)
    _check_decode(ga.kv4_attention(q, cache, table, lengths), q, kv, d, "f16")


@pytest.mark.parametrize("d,per", [(64, 12), (128, 9), (128, 16), (256, 5), (256, 11)])
def test_decode_join_many_units(d, per):
    """past 256 units the blocks have 4 waves: long sequences among them are shared all the same"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d + per)
    lens = rng.integers(0, 40, 140)
    lens[[3, 70, 139]] = 6000, 1500, 20000
    cache, table, lengths, kv = _paged(rng, lens.tolist(), 2, d, 16, 64, "bf16")
    q = _randn(rng, len(lens), 2 * per, d, dtype="bf16")
    _check_decode(ga.kv4_attention(q, cache, table, lengths), q, kv, 64, "bf16")


# ---------------------------------------------------------------- inside torch.compile

def test_compiled_caller():
    """a compiled function around the calls breaks its graph at them and gives what it gives uncompiled"""
    from grinqh import attention as ga
    rng = np.random.default_rng(31)
    cache, table, lengths, kv = _paged(rng, [3000, 40], 2, 64, 16, 64, "f16")
    x, ends = _randn(rng, 90, 8, 64), _dev([0, 30, 90])
    slots = torch.arange(90).cuda() - 1
    fresh = ga.kv4_cache(8, 2, 64)

    def layer(x, q):
        y = x * 0.5
        a = ga.prompt_attention(y[:, :4], y[:, 4:6], y[:, 6:], ends) + 1.0
        ga.kv4_store(fresh, y[:, 4:6], y[:, 6:], slots)
        k, v = ga.kv4_load(fresh, slots)
        return a, k + 1.0, v + 1.0, ga.kv4_attention(q + 1.0, cache, table, lengths) * 2.0

    compiled = torch.compile(layer, backend="eager")
    for i in range(3):
        q = _randn(rng, 2, 4, 64)
        for a, b in zip(compiled(x + i, q), layer(x + i, q)):
            assert torch.equal(a, b)
