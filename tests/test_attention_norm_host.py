"""The bound on the norm of an attention's error (_attention_norm.py) sees what it is for: mistakes planted in the oracle,
on the inputs of the GPU tests, are refused, and the arithmetic that the kernels state is accepted."""
import numpy as np
import pytest
import torch

from _attention_norm import close, definition, kept, worst


def _inputs(tokens, rows, d, per=2, group=32):
    rng = np.random.default_rng(tokens + d)
    k, v = (torch.from_numpy(rng.standard_normal((tokens, 1, d)).astype(np.float32)).half() for _ in range(2))
    k[:, :, ::17] += 6.0
    q = torch.from_numpy(rng.standard_normal((rows, per, d)).astype(np.float32)).half()
    return q.double(), kept(k, group), kept(v, d)


def _tile(at, factor):
    def weigh(p):
        p = p.clone()
        p[..., at:at + 64] *= factor
        return p
    return weigh


CASES = [(9000, 300, 64), (9000, 300, 128), (9000, 60, 256), (2777, 40, 128), (413, 150, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,rows,d", CASES)
def test_planted_mistakes_are_seen(tokens, rows, d, dtype):
    q, k, v = _inputs(tokens, rows, d)
    want = definition(q, k, v)
    seen_last = torch.cat((torch.zeros_like(k[:1]), k))[:-1], torch.cat((torch.zeros_like(v[:1]), v))[:-1]
    early, late = tokens // 64 // 3 * 64, (tokens - rows) // 64 * 64
    wrong = {
        "zeros": torch.zeros_like(want),
        "rows in reverse": want.flip(0),
        "a head's results in another": want.flip(1),
        "tokens behind the row's own": definition(torch.cat((q, q[-1:])), torch.cat((k, k[-1:])),
                                                  torch.cat((v, v[-1:])))[1:],
        "one token fewer": definition(q, *seen_last),
        "half of the tokens": definition(q, k, v, weigh=lambda p: torch.cat((p[..., :tokens // 2],
                                                                             0 * p[..., tokens // 2:]), -1)),
        "an early tile lost": definition(q, k, v, weigh=_tile(early, 0.0)),
        "a late tile lost": definition(q, k, v, weigh=_tile(late, 0.0)),
        "a tile twice": definition(q, k, v, weigh=_tile(early, 2.0)),
        "a part in the wrong unit": definition(q, k, v, weigh=lambda p: torch.cat((p[..., :early] * 1.25,
                                                                                  p[..., early:]), -1)),
    }
    for name, out in wrong.items():
        assert not close(out, want, dtype), name


@pytest.mark.parametrize("tokens,rows,d", CASES)
def test_stated_roundings_are_accepted(tokens, rows, d):
    """keys, values and weights in fp16, weights summed as rounded, results in the tensors' type"""
    q, k, v = _inputs(tokens, rows, d)
    want = definition(q, k, v)
    half = lambda x: x.half().double()  # noqa: E731
    out = definition(q, half(k), half(v), weigh=lambda p: half(p * 256.0))
    assert close(out.half(), want, "f16") and close(out.bfloat16(), want, "bf16")
    assert bool(((out.half().double() - want).pow(2).sum(-1).sqrt() <= worst(q, k, v, "f16", want)).all())
    assert not close(want * (1 + 1.1e-3), want, "f16") and not close(want * (1 + 3.3e-3), want, "bf16")
