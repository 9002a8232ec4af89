"""CPU checks of the serving operators' host path (grinqh/attention.py): what
is refused before anything is launched, which device the library is called on,
and the C entry points' own checks."""
import pytest
import torch

from grinqh import _lib
from grinqh import attention as ga
from test_attention_edges_host import Devices, _second

I32 = torch.int32


def _args(**changed):
    a = dict(q=_second(6, 8, 128), cache=_second(4, 2, 1, 2176, dtype=torch.uint8), table=_second(3, 5, dtype=I32),
             lengths=_second(3, dtype=I32), ends=_second(4, dtype=I32), counts=_second(3, dtype=I32),
             free=_second(9, dtype=I32), free_count=_second(1, dtype=I32), summary=_second(4, 2, 144, dtype=torch.int8),
             starts=_second(3, dtype=I32), page=16, tokens=6, count=4)
    assert set(changed) <= set(a)
    a.update(changed)
    return a


def _append(a):
    return ga.kv4_append(a["table"], a["lengths"], a["counts"], a["free"], a["free_count"], a["page"], a["tokens"])


def _chunk(a):
    return ga.kv4_chunk_attention(a["q"], a["cache"], a["table"], a["lengths"], a["ends"])


def _summarize(a):
    return ga.kv4_summarize(a["cache"], a["summary"], a["table"], a["starts"], a["lengths"])


def _select(a):
    return ga.kv4_select(a["q"][:3], a["summary"], a["table"], a["lengths"], a["page"], a["count"])


@pytest.fixture
def devices(monkeypatch):
    d = Devices(monkeypatch, ga)
    for cached in (ga._chunk_workspace_bytes, ga._workspace_bytes):
        cached.cache_clear()
    yield d
    for cached in (ga._chunk_workspace_bytes, ga._workspace_bytes):
        cached.cache_clear()
    ga._WORKSPACES._bufs.clear()


@pytest.mark.parametrize("current", [0, 1])
def test_calls_run_on_the_tensors_device(devices, monkeypatch, current):
    devices.current = current
    a = _args()
    _append(a)
    _chunk(a)
    _summarize(a)
    _select(a)
    ga.kv4_attention(a["q"][:3], a["cache"], _second(3, 2, 4, dtype=I32), a["lengths"])
    assert devices.calls == [(f"grinqh_{n}", 1) for n in ("kv4_append", "kv4_chunk_attention", "kv4_summarize",
                                                         "kv4_select", "kv4_attention_selected")]
    assert devices.current == current


BAD_Q = [dict(q=_second(6, 8, 64)), dict(q=_second(6, 7, 128)), dict(q=_second(6, 0, 128)), dict(q=_second(6, 1024)),
         dict(q=torch.zeros((6, 8, 128), dtype=torch.float16)), dict(q=_second(6, 8, 128, dtype=torch.float32)),
         dict(q=_second(6, 8, 128).requires_grad_())]
BAD_TABLE = [dict(table=_second(3, 5, dtype=torch.int64)), dict(table=_second(2, 5, dtype=I32)),
             dict(table=_second(15, dtype=I32)), dict(table=torch.zeros((3, 5), dtype=I32))]
BAD_LENGTHS = [dict(lengths=_second(3, dtype=torch.int64)), dict(lengths=_second(3, 1, dtype=I32)),
               dict(lengths=torch.zeros(3, dtype=I32))]
BAD_CACHE = [dict(cache=_second(4, 2, 1, 2175, dtype=torch.uint8)), dict(cache=_second(4, 0, 1, 2176, dtype=torch.uint8)),
             dict(cache=_second(4, 2, 2176, dtype=torch.uint8)), dict(cache=_second(4, 2, 1, 2176, dtype=torch.int8)),
             dict(cache=torch.zeros((4, 2, 1, 2176), dtype=torch.uint8))]
BAD_SUMMARY = [dict(summary=_second(4, 2, 143, dtype=torch.int8)), dict(summary=_second(4, 2, 144, dtype=torch.uint8)),
               dict(summary=_second(4, 144, dtype=torch.int8)), dict(summary=_second(4, 2, 160, dtype=torch.int8)[:, :, 16:]),
               dict(summary=_second(4, 0, 144, dtype=torch.int8)), dict(summary=torch.zeros((4, 2, 144), dtype=torch.int8))]


@pytest.mark.parametrize("call,bad", (
    [(_chunk, x) for x in BAD_Q + BAD_TABLE + BAD_LENGTHS + BAD_CACHE + [
        dict(ends=_second(4, dtype=torch.int64)), dict(ends=_second(0, dtype=I32)), dict(ends=_second(5, dtype=I32)),
        dict(ends=_second(2, 2, dtype=I32)), dict(lengths=_second(4, dtype=I32))]]
    + [(_append, x) for x in BAD_TABLE + BAD_LENGTHS + [
        dict(counts=_second(4, dtype=I32)), dict(counts=_second(3, dtype=torch.int64)),
        dict(free=_second(9, dtype=torch.int64)), dict(free=_second(3, 3, dtype=I32)),
        dict(free_count=_second(2, dtype=I32)), dict(free_count=_second(1, dtype=torch.int64)),
        dict(page=24), dict(page=8), dict(page=0), dict(page=-16), dict(tokens=-1), dict(tokens=1 << 23),
        # the table is written in place
        dict(table=_second(5, 3, dtype=I32).t()), dict(table=_second(1, 5, dtype=I32).expand(3, 5)),
        dict(table=_second(7, dtype=I32).as_strided((3, 5), (1, 1)))]]
    + [(_summarize, x) for x in BAD_TABLE + BAD_LENGTHS + BAD_CACHE + BAD_SUMMARY + [
        dict(starts=_second(2, dtype=I32)), dict(starts=_second(3, dtype=torch.int64)),
        dict(summary=_second(5, 2, 144, dtype=torch.int8)), dict(summary=_second(4, 1, 144, dtype=torch.int8)),
        dict(summary=_second(4, 2, 80, dtype=torch.int8))]]
    + [(_select, x) for x in BAD_Q + BAD_TABLE + BAD_LENGTHS + BAD_SUMMARY + [
        dict(count=1), dict(count=0), dict(count=-3), dict(page=24), dict(page=0),
        dict(summary=_second(4, 2, 80, dtype=torch.int8))]]))
def test_refused(devices, call, bad):
    with pytest.raises((ValueError, TypeError)):
        call(_args(**bad))
    assert devices.calls == []


def test_tables_per_head_are_checked(devices):
    a = _args()
    for table in (_second(3, 3, 4, dtype=I32), _second(2, 2, 4, dtype=I32), _second(3, 2, 4, dtype=torch.int64),
                  torch.zeros((3, 2, 4), dtype=I32), _second(3, 2, 4, 1, dtype=I32)):
        with pytest.raises(ValueError):
            ga.kv4_attention(a["q"][:3], a["cache"], table, a["lengths"])
    assert devices.calls == []


def test_host_tensors_are_refused():
    t = torch.zeros((2, 2), dtype=I32)
    with pytest.raises(ValueError, match="HIP device"):
        ga.kv4_append(t, t[0], t[0], t[0], t[0, :1], 16, 4)
    with pytest.raises(ValueError, match="HIP device"):
        ga.kv4_select(torch.zeros((2, 4, 64)).half(), torch.zeros((3, 2, 80), dtype=torch.int8), t, t[0], 16, 2)


# ---------------------------------------------------------------- C entry points

P = 1 << 12  # an address that is never read: every call below ends before a launch


def _c(name, *args):
    return getattr(_lib.load_library(), name)(*args)


def _with(args, **changed):
    names, values = zip(*args)
    out = dict(args)
    assert set(changed) <= set(names)
    out.update(changed)
    return [out[n] for n in names]


APPEND = [("table", P), ("stride", 4), ("width", 4), ("page", 16), ("lengths", P), ("counts", P), ("seqs", 3),
          ("free", P), ("size", 9), ("free_count", P), ("tokens", 6), ("slots", P), ("positions", P), ("ends", P),
          ("new_lengths", P), ("new_count", P), ("stream", None)]
CHUNK = [("q", P), ("q_token", 1024), ("q_head", 128), ("tokens", 6), ("heads", 8), ("cache", P), ("pages", 4),
         ("kv_heads", 2), ("page", 16), ("d", 128), ("group", 128), ("table", P), ("stride", 5), ("width", 5),
         ("lengths", P), ("ends", P), ("seqs", 3), ("scale", 1.0), ("out", P), ("dtype", 0), ("ws", None), ("bytes", 0),
         ("stream", None)]
SUMMARIZE = [("cache", P), ("pages", 4), ("kv_heads", 2), ("page", 16), ("d", 128), ("group", 128), ("summary", P),
             ("table", P), ("stride", 5), ("width", 5), ("starts", P), ("lengths", P), ("seqs", 3), ("stream", None)]
SELECT = [("q", P), ("q_token", 1024), ("q_head", 128), ("seqs", 3), ("heads", 8), ("summary", P), ("pages", 4),
          ("kv_heads", 2), ("page", 16), ("d", 128), ("table", P), ("stride", 5), ("width", 5), ("lengths", P),
          ("count", 4), ("selected", P), ("new_lengths", P), ("dtype", 0), ("ws", None), ("bytes", 0), ("stream", None)]


@pytest.mark.parametrize("name,args,bad", (
    [("kv4_append", APPEND, x) for x in (
        dict(page=24), dict(page=0), dict(page=-16), dict(width=-1), dict(width=1 << 28), dict(seqs=-1),
        dict(seqs=(1 << 20) + 1), dict(size=-1), dict(size=1 << 31), dict(tokens=-1), dict(tokens=1 << 23),
        dict(stride=3), dict(free_count=None), dict(ends=None), dict(new_count=None), dict(free=None), dict(slots=None),
        dict(positions=None), dict(lengths=None), dict(counts=None), dict(new_lengths=None), dict(table=None))]
    + [("kv4_chunk_attention", CHUNK, x) for x in (
        dict(dtype=2), dict(heads=7), dict(heads=0), dict(kv_heads=0), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=float("inf")), dict(scale=float("nan")), dict(seqs=-1), dict(seqs=(1 << 20) + 1), dict(tokens=-1),
        dict(tokens=1 << 30), dict(width=-1), dict(width=1 << 28), dict(d=96), dict(group=48), dict(group=256),
        dict(page=24), dict(pages=-1), dict(cache=None), dict(cache=P + 16), dict(q=None), dict(q=P + 2), dict(q_token=4),
        dict(q_head=-128), dict(q_token=(1 << 23) + 8), dict(ends=None), dict(lengths=None), dict(out=None),
        dict(out=P + 8), dict(table=None))]
    + [("kv4_summarize", SUMMARIZE, x) for x in (
        dict(kv_heads=0), dict(page=24), dict(d=96), dict(group=256), dict(pages=-1), dict(cache=None), dict(summary=None),
        dict(summary=P + 8), dict(table=None), dict(width=-1), dict(width=1 << 28), dict(starts=None), dict(lengths=None),
        dict(seqs=-1), dict(seqs=(1 << 20) + 1), dict(seqs=1 << 20, width=1 << 11))]
    + [("kv4_select", SELECT, x) for x in (
        dict(dtype=2), dict(heads=7), dict(kv_heads=0), dict(seqs=-1), dict(seqs=(1 << 20) + 1), dict(page=24), dict(d=96),
        dict(width=-1), dict(width=1 << 28), dict(count=1), dict(count=1 << 28), dict(pages=-1), dict(q=None),
        dict(q=P + 2), dict(q_head=4), dict(summary=None), dict(summary=P + 8), dict(table=None), dict(lengths=None),
        dict(selected=None), dict(new_lengths=None))]))
def test_c_entry_points_refuse(name, args, bad):
    assert _c(f"grinqh_{name}", *_with(args, **bad)) == _lib.GRINQH_ERR_INVALID


def test_c_entry_points_want_their_workspace():
    lib = _lib.load_library()
    need = lib.grinqh_kv4_chunk_attention_workspace_bytes(6, 3, 8, 2, 128, 4096 * 16)
    assert need > 1 << 17
    for ws, n in ((None, 0), (P, need - 1), (P + 16, need)):
        assert _c("grinqh_kv4_chunk_attention", *_with(CHUNK, width=4096, ws=ws, bytes=n)) == _lib.GRINQH_ERR_WORKSPACE
    need = lib.grinqh_kv4_select_workspace_bytes(3, 2, 4096, 4)
    assert need == 3 * 2 * 4096 * 4
    for ws, n in ((None, 0), (P, need - 1), (P + 16, need)):
        assert _c("grinqh_kv4_select", *_with(SELECT, width=4096, ws=ws, bytes=n)) == _lib.GRINQH_ERR_WORKSPACE


def test_nothing_to_do_needs_nothing():
    ok = _lib.GRINQH_OK
    assert _c("grinqh_kv4_chunk_attention", *_with(CHUNK, tokens=0, q=None, out=None, ends=None)) == ok
    assert _c("grinqh_kv4_summarize", *_with(SUMMARIZE, seqs=0, table=None, starts=None, lengths=None, summary=None)) == ok
    assert _c("grinqh_kv4_summarize", *_with(SUMMARIZE, pages=0, cache=None, summary=None)) == ok
    assert _c("grinqh_kv4_select", *_with(SELECT, seqs=0, q=None, table=None)) == ok


@pytest.mark.parametrize("tokens,seqs,heads,kv_heads,d,capacity", [
    (1, 1, 32, 8, 128, 512), (64, 16, 32, 8, 128, 2048), (543, 32, 32, 8, 128, 2560), (2048, 1, 32, 8, 128, 32768),
    (8192, 4, 64, 8, 128, 131072), (100000, 1, 128, 1, 64, 200000), (5, 4000, 64, 8, 256, 1 << 20), (7, 0, 4, 4, 64, 0)])
def test_workspaces_stay_small(tokens, seqs, heads, kv_heads, d, capacity):
    """what runs leave in the workspace is bounded by the card's blocks, whatever the batch"""
    n = _lib.load_library().grinqh_kv4_chunk_attention_workspace_bytes(tokens, seqs, heads, kv_heads, d, capacity)
    assert 0 <= n <= (1 << 17) + 2 * (512 * 16 * (d + 2) * 4 + 256 * 256 * (d + 2) * 4)
    if capacity <= 512:
        assert n == 0
