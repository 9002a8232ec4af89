"""CPU checks of the workspaces that captured attention calls take (grinqh/attention.py): one per capture and stream, its
counters cleared when it is made, and never an eager call's."""
import pytest
import torch

from grinqh import _lib
from grinqh import attention as ga
from test_attention_edges_host import Devices, _second

I32 = torch.int32


class Library:
    """records each call's workspace; ``capture`` is the capture that the stream takes part in, ``need`` what a call wants"""

    def __init__(self):
        self.capture, self.need, self.used = 0, 1 << 18, []

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            return lambda *args: self.need
        assert name in ("grinqh_kv4_attention", "grinqh_kv4_attention_selected", "grinqh_kv4_chunk_attention")

        def call(*args):
            self.used.append(args[-3:-1])  # workspace, bytes
            return 0
        return call

    def grinqh_capture_id(self, stream):
        return self.capture


@pytest.fixture
def library(monkeypatch):
    Devices(monkeypatch, ga)
    lib = Library()
    monkeypatch.setattr(_lib, "load_library", lambda: lib)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: lib.capture != 0)

    def clear():
        ga._workspace_bytes.cache_clear()
        ga._chunk_workspace_bytes.cache_clear()
        ga._WORKSPACES._bufs.clear()
    clear()
    yield lib
    clear()
    ga._GRAPH_WORKSPACES._bufs.clear()


def _calls():
    cache, table, lengths = _second(4, 2, 1, 2176, dtype=torch.uint8), _second(3, 5, dtype=I32), _second(3, dtype=I32)
    ga.kv4_attention(_second(3, 8, 128), cache, table, lengths)
    ga.kv4_attention(_second(3, 8, 128), cache, _second(3, 2, 4, dtype=I32), lengths)
    ga.kv4_chunk_attention(_second(6, 8, 128), cache, table, lengths, _second(4, dtype=I32))


def test_each_capture_has_a_workspace_of_its_own(library):
    taken = []
    for capture in (0, 7, 8, 0, 9):
        library.capture, library.used = capture, []
        _calls()
        taken.append(library.used)
        assert len(library.used) == 3 and len(set(library.used)) == 1  # shared within
        assert library.used[0][1] >= library.need
    eager, first, second, again, third = (x[0][0] for x in taken)
    assert again == eager and eager not in (first, second, third) and first != second != third


def test_counters_are_cleared_and_stay_with_the_capture(library, monkeypatch):
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(1))
    library.capture = 5
    _calls()
    (capture, ws), = ga._GRAPH_WORKSPACES._bufs.values()
    assert capture == 5 and ws.data_ptr() == library.used[0][0]
    assert not ws[:_lib.KV4_COUNTER_BYTES].any() and bool(ws[_lib.KV4_COUNTER_BYTES:].all())
    ws[:8] = 3
    _calls()
    assert bool((ws[:8] == 3).all())  # a second call finds them as the first one left them
    ga._workspace_bytes.cache_clear()
    ga._chunk_workspace_bytes.cache_clear()
    library.need = 1 << 19
    _calls()
    assert library.used[-1][1] >= 1 << 19 and library.used[-1][0] != library.used[0][0]


def test_streams_of_one_capture_are_apart(library, monkeypatch):
    library.capture = 3
    for stream in (11, 12):
        monkeypatch.setattr(ga, "_stream", lambda device, stream=stream: stream)
        _calls()
    assert len(set(library.used)) == 2


def test_an_unknown_capture_shares_nothing(library, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    kept = []
    get = ga._GRAPH_WORKSPACES.get
    monkeypatch.setattr(ga._GRAPH_WORKSPACES, "get", lambda *a: kept.append(get(*a)) or kept[-1])
    _calls()
    assert len(set(library.used)) == 3


def test_no_workspace_where_nothing_is_split(library):
    library.need, library.capture = 0, 4
    _calls()
    assert library.used == [(None, 0)] * 3 and not ga._GRAPH_WORKSPACES._bufs


def test_the_counters_are_where_the_header_says():
    lib = _lib.load_library()
    assert lib.grinqh_kv4_attention_workspace_bytes(1, 8, 8, 64, 1 << 20) > _lib.KV4_COUNTER_BYTES
    text = open(__file__.replace("tests/test_attention_graphs_host.py", "include/grinqh.h")).read()
    assert f"#define GRINQH_KV4_COUNTER_BYTES ((size_t)1 << {_lib.KV4_COUNTER_BYTES.bit_length() - 1})" in text
