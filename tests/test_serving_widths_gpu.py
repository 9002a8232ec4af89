"""kv4_select at the table widths where another kernel takes over, beside the ones below and above."""
import numpy as np
import pytest
import torch

import test_serving_gpu as serving

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


@pytest.mark.parametrize("width", [511, 512, 513, 1023, 1024, 1025, 1100, 2048])
@pytest.mark.parametrize("count", [2, 17, 700])
@pytest.mark.parametrize("dtype,d,per", [("f16", 128, 4), ("bf16", 64, 17), ("bf16", 256, 1)])
def test_select_at_changes_of_kernel(width, count, dtype, d, per):
    rng = np.random.default_rng(width + count + d)
    pages, hkv, lens = 300, 2, [width * 16, width * 16 - 17, 16 * min(count, width), 5, 0, width * 8]
    summary = serving._random_summary(rng, pages, hkv, d)
    q = serving._randn(rng, len(lens), hkv * per, d, dtype=dtype)
    table = rng.integers(0, pages, (len(lens), width))   # pages several times: equal scores
    serving._check_select(rng, q, summary, table, lens, 16, count)


@pytest.mark.parametrize("width", [1023, 1500, 2048])
def test_equal_scores_at_changes_of_kernel(width):
    """all alike, and two different scores only: ties go to the page that comes first"""
    rng = np.random.default_rng(width)
    base = serving._random_summary(rng, width, 1, 64, spread=1)
    q = serving._randn(rng, 1, 4, 64)
    table = rng.permutation(width).reshape(1, -1)
    few = base.copy()
    few[:, 0, :64] = rng.integers(0, 2, (width, 1)).astype(np.int8)
    for summary in (np.repeat(base[:1], width, 0), few, np.zeros_like(base)):
        for count in (2, 3, 77, width - 1):
            serving._check_select(rng, q, summary, table, [width * 16], 16, count)
