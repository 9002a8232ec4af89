"""What the cache's pages hold behind a sequence's last token has no effect on its results, whatever the bytes."""
import numpy as np
import pytest
import torch

from test_attention_gpu import _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _pair(scale, low):
    """(scale, minimum) as the cache keeps them; as codes, its nibbles"""
    return int(np.array([scale, low], np.float16).view(np.int32)[0])


INF, NAN = float("inf"), float("nan")
# the largest code stands for what fp16 can round to infinity, or nearly; and for more, for infinities and NaN
PAIRS = [(2.0, 65504.0), (4.0, 65504.0), (-2.0, -65504.0), (-370.0, -60000.0), (370.0, 60000.0), (1.0, 65504.0),
         (4370.0, 0.0), (-4370.0, 0.0), (65504.0, 65504.0), (-65504.0, 65504.0), (8736.0, -65504.0), (INF, 1.0),
         (1.0, INF), (-INF, INF), (0.0, -INF), (NAN, 1.0), (1.0, NAN)]


@pytest.mark.parametrize("rows", [1, 3, 70, 300])
@pytest.mark.parametrize("d,group,dtype", [(64, 32, "f16"), (128, 128, "bf16"), (256, 64, "f16")])
def test_bytes_behind_the_last_token(rows, d, group, dtype):
    from grinqh import attention as ga
    rng = np.random.default_rng(d + rows)
    lens = [rows + 5, 331, 307]
    k, v = ([_randn(rng, n, 1, d, dtype=dtype) for n in lens] for _ in range(2))
    q = _randn(rng, 3 * rows, 4, d, dtype=dtype)
    lengths, ends = (torch.tensor(x, dtype=torch.int32).cuda() for x in (lens, [0, rows, 2 * rows, 3 * rows]))
    table = torch.from_numpy(rng.permutation(63).astype(np.int32)).view(3, 21).cuda()
    wide = torch.nn.functional.pad(table, (0, 8000), value=-1)
    words = torch.randint(-(1 << 31), 1 << 31, (63, 1, 1, ga.kv4_record_bytes(d, group) // 4), dtype=torch.int64)
    want = None
    for name, fill in [("zeros", 0)] + [(x, _pair(*x)) for x in PAIRS] + [("random", words.to(torch.int32).cuda())]:
        cache = ga.kv4_cache(63, 1, d, 16, group)
        cache.view(torch.int32).copy_(fill) if torch.is_tensor(fill) else cache.view(torch.int32).fill_(fill)
        for i, n in enumerate(lens):
            at = torch.arange(n).cuda()
            ga.kv4_store(cache, k[i], v[i], table[i, at // 16].long() * 16 + at % 16)
        outs = [ga.kv4_chunk_attention(q, cache, t, lengths, ends) for t in (table, wide)]
        if rows == 1:
            outs += [ga.kv4_attention(q, cache, t, lengths) for t in (table, wide)]
        want = outs if want is None else want
        for out, clean in zip(outs, want):
            assert bool(clean.isfinite().all()) and torch.equal(out, clean), name
