"""The decoder example's steps over selected pages and with drafted tokens
(examples/decoder_attention.py): selecting every page changes nothing, and a
draft of several tokens at once agrees with the same tokens one by one."""
import pytest
import torch

from test_attention_example_gpu import _decoder

pytestmark = pytest.mark.gpu


def _started(lens, seed=5):
    model = _decoder()
    g = torch.Generator(device="cuda").manual_seed(seed)
    model.admit(len(lens))
    model.prompt(torch.randn((sum(lens), 512), generator=g, device="cuda").half(), lens)
    return model, g


def test_step_over_selected_pages():
    lens = [130, 100, 177]
    model, g = _started(lens)
    x = torch.randn((3, 512), generator=g, device="cuda").half()
    every = model.step(x, select=16)  # as many as there are
    again, _ = _started(lens)
    assert torch.equal(every, again.step(x))
    some, _ = _started(lens)
    out = some.step(x, select=4)
    assert bool(out.isfinite().all()) and not torch.equal(out, every)


def test_draft_agrees_with_single_tokens():
    """The kernels differ by their roundings (a few 2^-11 per layer) and by codes of the new tokens that these flip
    (half a scale in one channel, weighted by one key in the context's hundred), as between the step and the prompt path."""
    lens = [130, 100, 177]
    one, g = _started(lens)
    x = torch.randn((3, 4, 512), generator=g, device="cuda").half()
    single = torch.stack([one.step(x[:, i].contiguous()) for i in range(4)], 1)
    many, _ = _started(lens)
    draft = many.extend(x.flatten(0, 1), [4, 4, 4]).view(3, 4, 512)
    assert many.lengths.tolist() == one.lengths.tolist() == [n + 4 for n in lens]
    rms = float(single.float().pow(2).mean().sqrt())
    assert float((single.float() - draft.float()).abs().max()) <= 2.0 ** -5 * rms
