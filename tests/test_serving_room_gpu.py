"""kv4_append where pages run out: how a caller sees it, and that the call made again finds room for everything."""
import numpy as np
import pytest
import torch

import _attention_norm as norm
import test_serving_gpu as serving
from test_attention_example_gpu import _decoder
from test_attention_gpu import _randn

pytestmark = pytest.mark.gpu
_i32 = serving._i32


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _short(room):
    """a row of a sequence without a slot"""
    return bool((room.slots[:int(room.ends[-1])] < 0).any())


@pytest.mark.parametrize("more", ["pages", "fewer tokens"])
def test_the_call_made_again_finds_room(more):
    from grinqh import attention as ga
    rng = np.random.default_rng(2)
    page, news = 16, [40, 33, 70]
    cache = ga.kv4_cache(40, 2, 128, page)
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    free = torch.from_numpy(rng.permutation(40).astype(np.int32)).cuda()
    held = [_randn(rng, 1000, 2, 128) for _ in range(2)]
    given = _i32([0, 0, 0]), _i32([17, 30, 5]), free, _i32([11])
    room = ga.kv4_append(table, *given, page, 60)
    assert not _short(room)
    kv = [[x[a:b] for x in held] for a, b in ((0, 17), (17, 47), (47, 52))]
    ga.kv4_store(cache, *(x[:60] for x in held), room.slots)
    # 6 pages are left and 9 are needed
    lengths, count = room.lengths, room.free_count
    bad = ga.kv4_append(table, lengths, _i32(news), free, count, page, 150)
    assert _short(bad) and int(bad.free_count) == 0 and bool((table == -1).any())
    q = _randn(rng, 3, 8, 128)
    assert bool(ga.kv4_attention(q, cache, table, bad.lengths)[2].isnan().all())
    if more == "pages":
        free, count = torch.cat((free[:int(count)], free[11:])), count + 29
    else:
        news = [40, 33, 10]
    room = ga.kv4_append(table, lengths, _i32(news), free, count, page, 150)
    assert not _short(room) and room.lengths.tolist() == [17 + news[0], 30 + news[1], 5 + news[2]]
    used = [x for row, n in zip(table.tolist(), room.lengths.tolist()) for x in row[:-(-n // page)]]
    assert min(used) >= 0 and len(set(used)) == len(used)
    assert not set(used) & set(free[:int(room.free_count)].tolist())
    k, v = _randn(rng, 150, 2, 128), _randn(rng, 150, 2, 128)
    ga.kv4_store(cache, k, v, room.slots)
    at = 0
    for s, n in enumerate(news):
        kv[s] = [torch.cat((a, b[at:at + n])) for a, b in zip(kv[s], (k, v))]
        at += n
    rows = _randn(rng, 150, 8, 128)
    out = ga.kv4_chunk_attention(rows, cache, table, room.lengths, room.ends)
    norm.check(out, rows, kv, news, 128, "f16")
    norm.check(ga.kv4_attention(q, cache, table, room.lengths), q, kv, [1, 1, 1], 128, "f16")


def test_the_example_says_whether_all_have_room():
    model = _decoder()
    pages = len(model.free)
    g = torch.Generator(device="cuda").manual_seed(1)
    model.admit(3)
    model.free_count.fill_(12)
    h = lambda n: torch.randn((n, 512), generator=g, device="cuda").half()  # noqa: E731
    model.prompt(h(150), [40, 60, 50])
    assert model.all_have_room() and pages > 12
    before = model.lengths.clone(), model.free_count.clone()
    model.extend(h(60), [20, 20, 20])
    assert not model.all_have_room()
    left = int(before[1])
    model.free[left:left + 8] = model.free[12:20].clone()  # pages that came free meanwhile
    model.lengths, model.free_count = before[0], before[1] + 8
    out = model.extend(h(60), [20, 20, 20])
    assert model.all_have_room() and bool(out.isfinite().all())
