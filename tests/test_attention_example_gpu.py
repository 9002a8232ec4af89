"""The decoder example (examples/decoder_attention.py): prompts, single tokens
and a prompt behind a cached prefix through GRINQH linears and the 4-bit
cache.  The single-token path and the prompt path over loaded keys compute the
same attention from the same cache; they may differ by their roundings (a few
2^-11 per layer) and by codes of the new token that these flip (half a scale in
one channel, weighted by one key in the context's hundred)."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _decoder():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    from decoder_attention import Decoder
    return Decoder()


def test_step_agrees_with_extend():
    lens = [130, 100, 177]
    g = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randn((sum(lens), 512), generator=g, device="cuda").half()
    new = [torch.randn((3, 512), generator=g, device="cuda").half() for _ in range(3)]
    outs = []
    for kind in ("step", "extend"):
        model = _decoder()
        model.admit(3)
        first = model.prompt(h, lens)
        assert bool(first.isfinite().all())
        rows = []
        for x in new:
            rows.append(model.step(x) if kind == "step" else model.extend(x, [1, 1, 1]))
        assert model.lengths.tolist() == [n + 3 for n in lens]
        outs.append((first, torch.stack(rows).float()))
    (first, a), (again, b) = outs
    assert torch.equal(first, again)
    rms = float(a.pow(2).mean().sqrt())
    assert float((a - b).abs().max()) <= 2.0 ** -5 * rms


def test_extend_in_pieces():
    """a prompt in one piece and in two: the second piece sees the first as the cache keeps it, so that its rows differ
    by the keys' and values' 4 bits, and the first piece's not at all"""
    g = torch.Generator(device="cuda").manual_seed(6)
    h = torch.randn((180, 512), generator=g, device="cuda").half()
    whole, pieces = _decoder(), _decoder()
    whole.admit(1)
    pieces.admit(1)
    a = whole.prompt(h, [180])
    b = pieces.prompt(h[:100], [100])
    c = pieces.extend(h[100:], [80])
    assert float((a[:100] - b).abs().max()) <= 2.0 ** -7 * float(a.float().abs().max())
    rel = (a[100:].float() - c.float()).norm() / a[100:].float().norm()
    assert 0.0 < float(rel) < 0.2
