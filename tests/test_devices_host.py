"""CPU check of the linears' host path: every library call is made with the
tensors' GPU current, whichever was current before."""
import pytest
import torch

from grinqh import kernel, producer, utils
from test_attention_edges_host import Devices, _second


@pytest.mark.parametrize("current", [0, 1])
def test_linears_run_on_the_tensors_device(monkeypatch, current):
    x, wide = _second(3, 128), _second(3, 256)
    w, codes = _second(128, 64, dtype=torch.int8), _second(128, 64, dtype=torch.uint8)
    planes, scale = _second(128, 16, dtype=torch.int32), _second(1, 64)
    sigma, row, norm = _second(1, 128, dtype=torch.float32), _second(1, dtype=torch.int64), _second(128)
    for module in (utils, producer):
        devices = Devices(monkeypatch, module)
    devices.current = current
    args = (x, planes, scale, None, 8, 128, 16, [0.0] * 4)
    kernel.run_product(*args, "reference")
    producer.rmsnorm_sigma(x, norm)
    producer.silu_mul_sigma(wide)
    producer.gemv_batch_union_sigma(*args, sigma)
    utils.pack_planes(codes)
    utils.prepare_weight(w)
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a, **k: self)
    utils.unpack_planes(planes, row, utils.BitLevel.EIGHT_BIT, 16)
    utils.dequantize(planes, scale, 8, 128, 16)
    utils.grade(x, [0.0] * 4, 8)
    for key in [key for key in kernel._WORKSPACES._bufs if key[1] == 1]:
        del kernel._WORKSPACES._bufs[key]
    assert devices.calls == [(f"grinqh_{n}", 1) for n in (
        "gemm_or_gemv", "rmsnorm_sigma", "silu_mul_sigma", "gemv_batch_union_sigma", "pack_planes", "prepare_weight",
        "unpack_planes", "dequantize", "grade")]
    assert devices.current == current
