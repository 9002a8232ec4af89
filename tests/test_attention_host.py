"""CPU checks of the attention operators' host side: layout sizes, refusals of
the C entry points before anything is launched, workspace plans."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from grinqh import _lib
    return _lib.load_library()


@pytest.mark.parametrize("d,g,size", [(128, 128, 2176), (128, 32, 2368), (64, 64, 1152), (64, 32, 1216),
                                      (256, 256, 4224), (256, 32, 4672)])
def test_record_bytes(lib, d, g, size):
    from grinqh.attention import kv4_record_bytes
    assert kv4_record_bytes(d, g) == size == lib.grinqh_kv4_record_bytes(d, g)


@pytest.mark.parametrize("d,g", [(96, 32), (128, 256), (128, 16), (128, 48), (0, 0), (64, 128)])
def test_record_bytes_refuses(lib, d, g):
    from grinqh.attention import kv4_record_bytes
    assert lib.grinqh_kv4_record_bytes(d, g) == 0
    with pytest.raises(ValueError):
        kv4_record_bytes(d, g)


def test_layouts_are_told_apart_by_their_records():
    from grinqh import attention as ga
    assert len(ga._LAYOUTS) == sum(g <= d for d in ga.HEAD_DIMS for g in ga.GROUPS)


@pytest.mark.parametrize("page", [0, 8, 24, 48, -16])
def test_cache_refuses_page_sizes(page):
    from grinqh import attention as ga
    with pytest.raises(ValueError):
        ga.kv4_cache(2, 2, 128, page, device="cpu")


def test_cache_shape():
    from grinqh import attention as ga
    assert ga.kv4_cache(3, 2, 128, 64, 32, device="cpu").shape == (3, 2, 4, 2368)


def test_host_tensors_are_refused():
    import torch
    from grinqh import attention as ga
    x = torch.zeros((2, 2, 128), dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ga.prompt_attention(x, x, x, i)
    with pytest.raises(ValueError):
        ga.kv4_load(ga.kv4_cache(1, 2, 128, device="cpu"), torch.zeros(2, dtype=torch.int64))


def test_c_entry_points_refuse(lib):
    """status 1 for every bad argument; pointers are never followed on the host"""
    p = ctypes.c_void_p(4096)
    bad_p = ctypes.c_void_p(4104)

    def store(k=p, kt=256, kh=128, tokens=2, cache=p, pages=2, heads=2, page=16, d=128, g=128, dt=0, slots=p):
        return lib.grinqh_kv4_store(k, kt, kh, p, 256, 128, slots, tokens, cache, pages, heads, page, d, g, dt, None)

    for kw in ({"k": bad_p}, {"k": None}, {"kt": 257}, {"kt": -8}, {"kh": 4}, {"kt": 1 << 24}, {"tokens": -1},
               {"cache": None}, {"cache": bad_p}, {"pages": -1}, {"heads": 0}, {"page": 24}, {"page": 48}, {"d": 96},
               {"g": 16}, {"dt": 2}, {"slots": None}):
        assert store(**kw) == 1, kw
    assert store(tokens=0) == 0 and store(pages=0, cache=None) == 0

    def attend(q=p, seqs=2, heads=8, kv=2, table=p, width=4, lengths=p, scale=0.1, out=p, dt=0, ws=None, n=0):
        return lib.grinqh_kv4_attention(q, 1024, 128, seqs, heads, p, 8, kv, 16, 128, 128, table, width, width, lengths,
                                        scale, out, dt, ws, n, None)

    for kw in ({"q": None}, {"q": bad_p}, {"seqs": -1}, {"heads": 7}, {"heads": 0}, {"kv": 0}, {"table": None},
               {"width": -1}, {"width": 1 << 30}, {"lengths": None}, {"scale": 0.0},
               {"scale": float("nan")}, {"scale": float("inf")}, {"out": None}, {"out": bad_p}, {"dt": 5}):
        assert attend(**kw) == 1, kw
    assert attend(seqs=0) == 0
    assert attend(width=10000) == 3  # no workspace
    need = lib.grinqh_kv4_attention_workspace_bytes(2, 8, 2, 128, 160000)
    assert need > 0
    assert attend(width=10000, ws=p, n=need - 1) == 3
    assert attend(width=10000, ws=bad_p, n=need) == 3

    def prompt(q=p, k=p, kt=256, heads=8, kv=2, d=128, rows=5, keys=5, ends=p, seqs=1, scale=0.1, out=p, dt=0):
        return lib.grinqh_prompt_attention(q, 1024, 128, k, kt, 128, p, 256, 128, ends, p, seqs, rows, keys, heads, kv,
                                           d, scale, out, dt, None)

    for kw in ({"q": None}, {"k": bad_p}, {"kt": 0}, {"kt": 120}, {"heads": 3}, {"kv": 0}, {"d": 80}, {"rows": -1}, {"keys": -1},
               {"rows": 1 << 31}, {"ends": None}, {"seqs": -1}, {"scale": -1.0}, {"out": None}, {"dt": 9}):
        assert prompt(**kw) == 1, kw
    assert prompt(rows=0) == 0


def test_workspace_query(lib):
    q = lib.grinqh_kv4_attention_workspace_bytes
    counters = 4 << 15
    assert q(1, 32, 8, 128, 1024) == 0          # one run of 32 steps
    assert q(1, 32, 8, 128, 1025) == counters + (8 + 8) * (4 * 128 + 32) * 4
    assert q(1, 32, 8, 128, 131072) == counters + (8 + 256) * (4 * 128 + 32) * 4
    assert q(1, 64, 1, 64, 131072) == counters + (4 + 256) * (16 * 64 + 32) * 4   # 4 tiles of 16 query heads
    assert q(5000, 32, 8, 128, 131072) == 0     # more units than counters: none is shared
    assert q(1024, 4, 1, 128, 131072) > 0 and q(1025, 4, 1, 128, 131072) == 0   # more sequences than a plan covers
    assert q(0, 32, 8, 128, 100) == 0 and q(1, 5, 2, 128, 100) == 0 and q(1, 4, 2, 128, 0) == 0
