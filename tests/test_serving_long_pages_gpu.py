"""The operators around the 4-bit cache with long pages: one page for a whole sequence, pages that end inside a tile's
neighbour, and means over more tokens than one block of sums."""
import numpy as np
import pytest
import torch

import _attention_norm as norm
import test_serving_gpu as serving
from test_attention_gpu import _randn

pytestmark = pytest.mark.gpu
_i32 = serving._i32


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


@pytest.mark.parametrize("page", [128, 512, 4096, 16384])
@pytest.mark.parametrize("d,group,dtype", [(64, 64, "f16"), (128, 32, "bf16")])
def test_steps(page, d, group, dtype):
    from grinqh import attention as ga
    rng = np.random.default_rng(page + d)
    hkv, per, lens = 2, 4, [9000, 127, 4097]
    pages = sum(-(-n // page) + 1 for n in lens)
    cache, width = ga.kv4_cache(pages, hkv, d, page, group), -(-9100 // page) + 1
    cache.fill_(0xFF)
    summary = ga.kv4_summary(cache)
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    free, count, lengths = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda(), _i32([pages]), _i32([0] * 3)
    kv = [(torch.zeros((0, hkv, d), dtype=torch.float16, device="cuda"),) * 2] * 3
    for news in (lens, [70, 1, 3], [1, 1, 1]):
        rows = sum(news) + 4
        k, v = (_randn(rng, rows, hkv, d, dtype=dtype) for _ in range(2))
        room = ga.kv4_append(table, lengths, _i32(news), free, count, page, rows)
        assert bool((room.slots[:sum(news)] >= 0).all())
        ga.kv4_store(cache, k, v, room.slots)
        ga.kv4_summarize(cache, summary, table, lengths, room.lengths)
        lengths, count, at = room.lengths, room.free_count, 0
        for i, n in enumerate(news):
            kv[i] = tuple(torch.cat((a.to(k.dtype), b[at:at + n])) for a, b in zip(kv[i], (k, v)))
            at += n
        if rows < 1000:
            q = _randn(rng, rows, hkv * per, d, dtype=dtype)
            out = ga.kv4_chunk_attention(q, cache, table, lengths, room.ends)
            norm.check(out, q, kv, news, group, dtype)
            assert not out[-4:].any()
    got, tab = summary.cpu().numpy(), table.cpu().numpy()
    for i, (k, _) in enumerate(kv):
        codes, steps = serving._summary_ref([k], [len(k)], group, page)[0]
        at = tab[i, :len(codes)]
        assert np.array_equal(got[at, :, :d], codes)
        assert np.array_equal(serving._steps(got[at], d), steps.astype(np.float32))
    q = _randn(rng, 3, hkv * per, d, dtype=dtype)
    for n in (2, 3, 5):
        serving._check_select(rng, q, got, tab, lengths.tolist(), page, n)
    selected, some = ga.kv4_select(q, summary, table, lengths, page, width)
    norm.check(ga.kv4_attention(q, cache, selected, some), q, kv, [1] * 3, group, dtype)
