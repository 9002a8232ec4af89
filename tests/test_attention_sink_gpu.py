"""One token that outweighs all others by far, with a value near zero, and many thousands of others whose small weights
make up a good part of the result.

Keys are the same in all channels, which the cache keeps exactly, so logits are what they are meant to be.  Results are
held to _attention_norm's bound and to what weights below fp16's normal range add: those are off by 2^-25 where the
largest is between 2^7 and 2^15, so at most by 2^-32 of the largest each."""
import numpy as np
import pytest
import torch

import _attention_norm as norm
from test_attention_gpu import DT, U, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


TAILS = [(32768, 17.2, 0.05), (32768, 17.2, 0.0), (60000, 17.5, 0.3), (9000, 16.5, 1.0)]


def _tokens(tail, lower, spread, d, at, dtype, seed):
    """keys and values of `tail` tokens and of one whose logit is `lower` nats higher, at place `at`; queries are ones"""
    rng = np.random.default_rng(seed)
    z = -lower + spread * rng.standard_normal(tail + 1)
    z[at] = 0.0
    k = torch.from_numpy((z / d ** 0.5).astype(np.float32)).to(DT[dtype]).cuda().view(-1, 1, 1).repeat(1, 1, d)
    v = _randn(rng, tail + 1, 1, d) + 0.5 + _randn(rng, d)  # channels of different means
    v[at] *= 0.02 / v[at].abs().mean()
    return k, v.to(DT[dtype])


def _held(out, q, k, v, dtype, more=0.0):
    want = norm.definition(q, k, v)
    size = want.pow(2).sum(-1).sqrt().mean()
    below = len(v) * 2.0 ** -32 * (v.pow(2).sum((1, 2)).mean().sqrt() + size)
    err = (out.double().cpu() - want).pow(2).sum(-1).sqrt()
    assert float((err / size).max()) <= norm.BOUND[dtype] + more + float(below / size), float((err / size).max())


@pytest.mark.parametrize("tail,lower,spread", TAILS)
@pytest.mark.parametrize("rows", [1, 2, 300])
@pytest.mark.parametrize("d,dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
def test_cached_tokens(tail, lower, spread, rows, d, dtype):
    """kv4_attention (one row), and both kernels of kv4_chunk_attention, whole units, runs and pieces"""
    from grinqh import attention as ga
    for at in (0, tail // 2, tail - rows):
        k, v = _tokens(tail, lower, spread, d, at, dtype, tail)
        pages = -(-len(k) // 16)
        cache = ga.kv4_cache(pages, 1, d)
        ga.kv4_store(cache, k, v, torch.arange(len(k)).cuda())
        table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
        lengths, ends = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([len(k)], [0, rows]))
        q = torch.ones((rows, 4, d), dtype=DT[dtype], device="cuda")
        kept = norm.kept(k, d), norm.kept(v, d)
        outs = [ga.kv4_chunk_attention(q, cache, t, lengths, ends)
                for t in (table, torch.nn.functional.pad(table, (0, 8000), value=-1))]
        if rows == 1:
            outs.append(ga.kv4_attention(q, cache, table, lengths))
        if rows == 300:  # units enough for every block: none is split, and all tokens are beside the one
            n = 256
            out = ga.kv4_chunk_attention(q[:1].expand(n * rows, -1, -1), cache, table.expand(n, -1), lengths.expand(n),
                                         torch.arange(0, n * rows + 1, rows, dtype=torch.int32).cuda())
            outs += [out[:rows], out[-rows:]]
        for out in outs:
            _held(out, q, *kept, dtype)


@pytest.mark.parametrize("tail,lower,spread", TAILS)
@pytest.mark.parametrize("d,dtype", [(64, "f16"), (128, "f16"), (256, "f16"), (128, "bf16")])
def test_prompts(tail, lower, spread, d, dtype):
    """Rows behind a long run of keys.  A weight's rounding does not change the sum that divides it: tokens that weigh
    nearly the same are all off by the same 2^-11 or, of bf16 tensors, 2^-8."""
    from grinqh import attention as ga
    for rows, at in ((300, 0), (300, tail // 2), (1, 0), (40, tail - 40)):
        k, v = _tokens(tail, lower, spread, d, at, dtype, tail)
        ends, key_ends = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, rows], [0, len(k)]))
        q = torch.ones((rows, 2, d), dtype=DT[dtype], device="cuda")
        _held(ga.prompt_attention(q, k, v, ends, key_ends), q, k.double().cpu(), v.double().cpu(), dtype,
              more=U[dtype])


@pytest.mark.parametrize("power", range(20, 31))
@pytest.mark.parametrize("part", [1.0, 1.125, 1.5, 1.9375])
def test_logits_where_fp32_has_steps_of_1_to_64(power, part):
    """Logits of 2^23 to 2^34: the reference below the largest one is rounded, and the largest weight stays in range.  Two
    tokens' logits are the same and far above the others': the result is the mean of their values, each rounded to fp16
    once and the mean to bf16."""
    from grinqh import attention as ga
    rng = np.random.default_rng(power)
    n, rows = 200, 60
    k = (torch.from_numpy(rng.uniform(-0.5, 0.5, (n, 1, 1)).astype(np.float32)).half().cuda()).repeat(1, 1, 64)
    v = _randn(rng, n, 1, 64)
    k[7], k[131] = 1.0, 1.0
    cache = ga.kv4_cache(13, 1, 64)
    ga.kv4_store(cache, k, v, torch.arange(n).cuda())
    table = torch.nn.functional.pad(torch.arange(13, dtype=torch.int32).view(1, -1), (0, 8000), value=-1).cuda()
    q = torch.full((rows, 2, 64), part * 2.0 ** power, dtype=torch.bfloat16, device="cuda")
    out = ga.kv4_chunk_attention(q, cache, table, torch.tensor([n], dtype=torch.int32).cuda(),
                                 torch.tensor([0, rows], dtype=torch.int32).cuda()).double().cpu()
    a, b = norm.kept(v, 64)[[7, 131], 0]
    assert bool(((out - (a + b) / 2).abs() <= 2.0 ** -11 * (a.abs() + b.abs()) + 2.0 ** -8 * ((a + b) / 2).abs()).all())
