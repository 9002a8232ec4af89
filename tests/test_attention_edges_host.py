"""CPU checks of the attention operators' host path at its edges: which device
the library is called on, which inputs are copied or refused, what workspaces
cover."""
import pytest
import torch

from grinqh import _lib
from grinqh import attention as ga

SECOND = torch.device("cuda", 1)


class OnSecond(torch.Tensor):
    """A host tensor that says it is on the second GPU."""
    is_cuda = True
    device = SECOND


def _second(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnSecond)


class Devices:
    """Stands in for the current device and for the library; notes the device of every C call."""

    def __init__(self, monkeypatch, module):
        self.current, self.calls = 0, []
        here, empty = self, torch.empty

        class Guard:
            def __init__(self, device):
                self.device = device

            def __enter__(self):
                self.before, here.current = here.current, self.device.index

            def __exit__(self, *error):
                here.current = self.before

        class Library:
            def __getattr__(self, name):
                if name.endswith("bytes"):
                    return lambda *args: 1024
                return lambda *args: here.calls.append((name, here.current)) or 0

        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        for make in ("empty", "zeros"):
            original = getattr(torch, make)
            monkeypatch.setattr(torch, make, lambda *a, device=None, original=original, **k: original(*a, **k))
        monkeypatch.setattr(torch, "empty_like", lambda x, **k: empty(x.shape, dtype=x.dtype))
        monkeypatch.setattr(_lib, "load_library", lambda: Library())
        if hasattr(module, "_stream"):
            monkeypatch.setattr(module, "_stream", lambda device: 0)


@pytest.mark.parametrize("current", [0, 1])
def test_attention_runs_on_the_tensors_device(monkeypatch, current):
    cache, q, k = _second(2, 2, 1, 2176, dtype=torch.uint8), _second(3, 8, 128), _second(3, 2, 128)
    slots, lengths, table = (_second(*s, dtype=d) for s, d in (((3,), torch.int64), ((3,), torch.int32),
                                                             ((3, 4), torch.int32)))
    devices = Devices(monkeypatch, ga)
    devices.current = current
    ga._workspace_bytes.cache_clear()
    ga.kv4_store(cache, k, k, slots)
    ga.kv4_load(cache, slots)
    ga.kv4_attention(q, cache, table, lengths)
    ga.prompt_attention(q, k, k, lengths)
    ga._workspace_bytes.cache_clear()
    ga._WORKSPACES._bufs.clear()
    assert devices.calls == [(f"grinqh_{n}", 1) for n in ("kv4_store", "kv4_load", "kv4_attention", "prompt_attention")]
    assert devices.current == current


def _askew(x):
    """x [tokens, heads, d], called contiguous by torch, one element off the alignment that the kernels read"""
    return torch.empty(x.numel() + 1, dtype=x.dtype)[1:].view(x.shape).copy_(x)


def test_rows_are_copied_where_the_kernels_cannot_read_them():
    x = torch.randn((4, 3, 128)).half()
    wide = torch.randn((4, 1, 129)).half()
    cases = [_askew(x), _askew(x[:1]), wide[:, :, 1:], wide[:1, :, 1:], x[:1].as_strided((1, 3, 128), (3, 128, 1)),
             x[:1].as_strided((1, 3, 128), ((1 << 23) + 8, 128, 1)), x[:, :1].as_strided((4, 1, 128), (384, 5, 1)),
             x[:1].expand(4, -1, -1), x.as_strided((4, 3, 128), (64, 128, 1))]
    for y in cases:
        got, token, head = ga._rows(y, "x", y.device, y.dtype, 128)
        assert torch.equal(got, y) and got.data_ptr() % 16 == 0 and got.stride() == (token, head, 1)
        assert 128 <= token <= 1 << 23 and token % 8 == 0 and 0 <= head <= 1 << 23 and head % 8 == 0
    for y in (x, x[:, :2], x[::2], x.transpose(0, 1), x[:1].expand(4, -1, -1)):  # read in place
        assert ga._rows(y, "x", y.device, y.dtype)[0] is y


def test_tangents_are_refused():
    """a forward-mode dual does not require a gradient; its tangent must not be dropped in silence"""
    x = torch.randn((4, 3, 128)).half()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for y in (dual, dual[:, :2], dual[:1, 1:]):
            with pytest.raises(ValueError, match="tangent"):
                ga._rows(y, "q", x.device, x.dtype)
        assert ga._rows(x, "q", x.device, x.dtype)[0] is x

    def through(y):
        with pytest.raises(ValueError, match="tangent"):
            ga._rows(y, "q", x.device, x.dtype)
        return y * 2
    torch.func.jvp(through, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("heads,kv_heads,d,capacity", [(32, 8, 128, 8192), (2, 1, 64, 2048), (64, 8, 256, 1 << 20),
                                                       (40, 40, 64, 4096), (17, 1, 128, 1056), (128, 1, 64, 40000),
                                                       (8, 8, 128, 1024)])
def test_workspace_covers_all_smaller_batches(heads, kv_heads, d, capacity):
    ga._workspace_bytes.cache_clear()
    query = _lib.load_library().grinqh_kv4_attention_workspace_bytes
    most = 0
    for seqs in range(1, 4300):
        most = max(most, query(seqs, heads, kv_heads, d, capacity))
        assert ga._workspace_bytes(seqs, heads, kv_heads, d, capacity) == most
    assert (most > 0) == (capacity > 1024)
    assert ga._workspace_bytes(1 << 20, heads, kv_heads, d, capacity) == most
    ga._workspace_bytes.cache_clear()
